"""The end of a training step: gradient norm, clipping and the AdamW update
over all leaves of a scene at once (csrc/optim.cu).

The reference leaves the optimiser to its caller.  A caller of this package
has the gradients of a handful of large leaves (means, quaternions, scales,
opacities, SH coefficients) and of many small ones (camera poses), and these
functions take them all in one or two launches, without a host round trip:

  * `gradient_norm(grads)`: the global norm, and each tensor's if asked;
  * `clip_gradients_(grads, max_norm)`: scales the gradients in place so that
    their global norm is at most `max_norm`;
  * `adamw_update_(params, grads, exp_avgs, exp_avg_sqs, step, ...)`: the
    AdamW update, with the clipping coefficient applied on the way
    (`max_norm`), rows that no sensor saw left as they are (`row_mask`) and
    half-precision parameters kept beside 32-bit masters (`masters`);
  * `AdamW`: a `torch.optim.Optimizer` over these.

Tensors are float32, bfloat16 or float16 on one CUDA device; moments and
masters are float32.  Work is enqueued on the current stream and nothing is
read back.  Results do not depend on the run: sums are taken in an order that
goes by the tensors' sizes and addresses modulo 128 bytes.
"""
from __future__ import annotations

from collections.abc import Sequence

import torch

from ._native import _C


def gradient_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0, per_tensor: bool = False):
    """The norm of all elements of all `grads` as a 0-dim float32 tensor on
    their device; `norm_type` is 2, 1 or inf.  `per_tensor`: also a tensor
    with each one's norm.  Sums are held in 64 bits, so large and tiny
    gradients neither overflow nor vanish on the way; NaN and infinite
    elements show in the result.  A tensor with gaps or expanded dimensions is
    copied first.  The norm is taken outside autograd: nothing flows back
    through it, whether or not the gradients have a graph (`create_graph`)."""
    return _C.gradient_norm(grads, norm_type, per_tensor)


def clip_gradients_(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """Multiplies `grads` in place by min(1, max_norm / (norm + 1e-6)) and
    returns the norm that they had.  An infinite norm gives the factor 0, a
    NaN makes every gradient NaN.  The scaling is outside autograd: a graph
    that the gradients have knows nothing of it.  The tensors must be dense and
    may not share memory.  For the norm alone, without a limit, there is
    `gradient_norm`."""
    return _C.clip_gradients_(grads, max_norm, norm_type)


def adamw_step_counter(device, updates: int = 0) -> torch.Tensor:
    """The `step` of `adamw_update_`: the number of updates taken, which the
    call advances on the device, and a word that has to be zero between calls
    (the call's blocks count themselves in it), so that calls that share a
    counter follow one another on a stream.  Where they do not, updates may be
    counted wrongly; every element is still updated once by each."""
    return torch.tensor([updates, 0], dtype=torch.int64, device=device)


def adamw_update_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
                  exp_avg_sqs: Sequence[torch.Tensor], step: torch.Tensor, *, lr, betas=(0.9, 0.999), eps=1e-8,
                  weight_decay=0.0, max_norm: float | None = None, skip_nonfinite: bool = False,
                  masters: Sequence[torch.Tensor | None] | None = None,
                  row_mask: torch.Tensor | Sequence[torch.Tensor | None] | None = None) -> torch.Tensor | None:
    """One AdamW update of `params` in place, outside autograd.  With t the
    number of updates taken so far plus one (`step`, from
    `adamw_step_counter`):

        m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,
        w <- w - lr * weight_decay * w - lr * (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

    lr, eps, weight_decay and both betas are one value for all tensors or a
    list with one for each.  `max_norm`: g is the gradient clipped to that
    global 2-norm (`grads` themselves stay as they are).  `skip_nonfinite`: a
    norm that is NaN or infinite leaves parameters, moments and `step` as they
    were.  With either, the norm before clipping is returned.  `masters`:
    32-bit parameters that half-precision `params` are roundings of; both are
    written.  `row_mask` (bool, one entry for each row of dimension 0; one for
    all tensors or a list): rows with False keep parameter and moments; the
    norm is of all gradients, theirs too.

    Written tensors must be dense and may not share memory; moments and
    masters have their parameter's sizes and order of dimensions.  A gradient
    in another order is copied first.  Under graph capture the learning rate
    is the one at capture."""
    return _C.adamw_update_(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas[0], betas[1], eps, weight_decay,
                            max_norm, skip_nonfinite, masters, row_mask)


def _updates_of(state_dict: dict) -> int:
    """The number of updates behind a checkpoint's moments."""
    if "updates" in state_dict:
        return int(state_dict["updates"])
    counts = {int(s["step"]) if "step" in s else None for s in state_dict["state"].values() if s}
    if not counts:
        return 0
    if len(counts) > 1 or None in counts:
        raise ValueError("AdamW: the checkpoint has no number of updates that holds for all its parameters")
    return counts.pop()


class AdamW(torch.optim.Optimizer):
    """AdamW over `adamw_update_`: all parameter groups in one update.

    Group options: lr, betas, eps, weight_decay.  `max_norm` clips the global
    2-norm over all groups; `skip_nonfinite` passes over steps whose norm is
    NaN or infinite.  Half-precision parameters get float32 masters.  The
    number of updates is one counter on the device for all parameters, so a
    parameter added later starts at the common count.  `grad_norm`: the norm
    before clipping of the last `step`, on the device."""

    grad_norm: torch.Tensor | None = None

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 *, max_norm: float | None = None, skip_nonfinite: bool = False):
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("AdamW: lr, eps and weight_decay must not be negative, betas in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.max_norm = max_norm
        self.skip_nonfinite = skip_nonfinite
        self._step: torch.Tensor | None = None

    def _state(self, p: torch.Tensor) -> dict:
        s = self.state[p]  # what a checkpoint has left out begins here
        for k in ("exp_avg", "exp_avg_sq"):
            if k not in s:
                s[k] = torch.zeros_like(p, dtype=torch.float32)
        if p.dtype != torch.float32 and "master" not in s:
            s["master"] = p.detach().to(torch.float32, copy=True)
        return s

    @torch.no_grad()
    def step(self, closure=None, *, row_masks: dict | None = None):
        """Updates every parameter that has a gradient; returns the global
        gradient norm before clipping (None without `max_norm` and
        `skip_nonfinite`) or, given a `closure`, what that returns (the norm is
        in `grad_norm` either way).  `row_masks`: for a parameter, the rows to
        update; the others keep their values and moments."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.grad_norm = self._update(row_masks)
        return self.grad_norm if closure is None else loss

    def _update(self, row_masks: dict | None) -> torch.Tensor | None:
        params, grads, ms, vs, masters, masks = [], [], [], [], [], []
        lr, b1, b2, eps, decay = [], [], [], [], []
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                s = self._state(p)
                params.append(p)
                grads.append(p.grad)
                ms.append(s["exp_avg"])
                vs.append(s["exp_avg_sq"])
                masters.append(s.get("master"))
                masks.append(row_masks.get(p) if row_masks else None)
                lr.append(group["lr"])
                b1.append(group["betas"][0])
                b2.append(group["betas"][1])
                eps.append(group["eps"])
                decay.append(group["weight_decay"])
        if not params:
            return None
        if self._step is None:
            self._step = adamw_step_counter(params[0].device)
        return adamw_update_(params, grads, ms, vs, self._step, lr=lr, betas=(b1, b2), eps=eps, weight_decay=decay,
                             max_norm=self.max_norm, skip_nonfinite=self.skip_nonfinite,
                             masters=masters if any(m is not None for m in masters) else None,
                             row_mask=masks if row_masks else None)

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite,
                "_step": self._step}

    def state_dict(self) -> dict:
        """The count of updates is in it once for all (`updates`) and, for what
        keeps state and groups alone, with each parameter (`step`)."""
        d = super().state_dict()
        d["updates"] = 0 if self._step is None else int(self._step[0])
        d["state"] = {i: {**s, "step": torch.tensor(float(d["updates"]))} for i, s in d["state"].items()
                      if s}
        return d

    def load_state_dict(self, state_dict: dict) -> None:
        """Takes `state_dict` of this class, or of `torch.optim.AdamW` (and
        `torch.optim.Adam` without decay) if all its parameters have had the
        same number of updates, without `amsgrad` and `maximize`."""
        updates = _updates_of(state_dict)
        for group in state_dict["param_groups"]:
            for option in ("amsgrad", "maximize"):
                if group.get(option):
                    raise ValueError(f"AdamW: {option} is not supported")
            if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
                raise ValueError("AdamW: the checkpoint's weight decay goes through its gradients")
        super().load_state_dict({k: v for k, v in state_dict.items() if k != "updates"})
        # the base class casts state to its parameter's type: masters and moments stay in 32 bits
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, mine):
            if i in state_dict["state"]:
                self.state[p] = {k: v.to(device=p.device, dtype=torch.float32, copy=True)
                                 for k, v in state_dict["state"][i].items() if k != "step"}
        self._step = adamw_step_counter(mine[0].device, updates)
