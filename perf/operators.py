"""The gradient operators of a training step, as they are measured: the global
gradient norm over many tensors, clipping by it, and the AdamW update that
takes the clipped gradient.

`own` selects what `run` computes with: the plain form (elementary torch
operations in 32 bits) or xsimgs_b200's kernels.  A case is one of three sets
of tensors:

  rig     `n` cameras refined with the scene: eight small tensors
          (rotation, position, velocities, shutter times, intrinsics);
  scene   `n` Gaussians with SH degree `degree`: means, quaternions, scales,
          opacities, SH coefficients.  The gradient of a row that no view saw
          is zero; the others spread over several decades;
  bucket  `tensors` tensors of ragged sizes, `n` elements in all, laid one
          after another in a flat buffer without padding, as a bucketed
          gradient exchange leaves them.
"""
import math
import random

import torch

own = False

BETAS = (0.9, 0.999)
CLIP_EPS = 1e-6
START = 120  # updates taken before the measured one
RIG_WIDTHS = (4, 3, 3, 3, 2, 1, 1, 4)
SCENE_LR = (1.6e-4, 1e-3, 5e-3, 5e-2, 2.5e-3)
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _case(name, op, kind, n, degree=0, tensors=0, dtype="fp32", norm="2", per_tensor=False, limit="none", seen=1.0,
          row_mask=False, masters=False):
    c = dict(op=op, kind=kind, n=n, degree=degree, tensors=tensors, dtype=dtype, norm=norm, per_tensor=per_tensor,
             limit=limit, seen=seen, row_mask=row_mask, masters=masters)
    return dict(c, name=name) if name else c


def listed():
    return [
        # pose refinement of an eight-camera rig: 168 floats, all latency
        _case("norm_rig8", "norm", "rig", 8),
        # the log line of a one-million-Gaussian scene: total and one norm for each leaf
        _case("norm_scene1m_each", "norm", "scene", 1_000_000, degree=3, per_tensor=True, seen=0.4),
        # largest gradient entry of a half-precision network's bucket, each tensor's own too
        _case("norm_bucket160m_inf", "norm", "bucket", 160_000_000, tensors=311, dtype="bf16", norm="inf",
              per_tensor=True),
        # clipping the small scene (10 k Gaussians, flat colour)
        _case("clip_scene10k", "clip", "scene", 10_000, limit="over", seen=0.9),
        # an odd-sized scene whose norm is within the limit: nothing has to be scaled, as in most steps
        _case("clip_scene499979_in", "clip", "scene", 499_979, degree=2, limit="in", seen=0.4),
        # half-precision bucket with odd offsets
        _case("clip_bucket90m", "clip", "bucket", 90_000_001, tensors=201, dtype="bf16", limit="over"),
        # the six-view rig's scene (2 M Gaussians, SH degree 3): larger than the L2
        _case("clip_scene2m", "clip", "scene", 2_000_000, degree=3, limit="over", seen=0.6),
        # pose refinement's update
        _case("adamw_rig6", "adamw", "rig", 6),
        # the small scene's whole step: norm, clipping and update
        _case("adamw_scene10k_clip", "adamw", "scene", 10_000, limit="over", seen=0.9),
        # one view's step: only the Gaussians that it saw are updated
        _case("adamw_scene1m_rows", "adamw", "scene", 1_000_000, degree=3, seen=0.35, row_mask=True),
        # half-precision parameters and gradients over 32-bit masters, clipped
        _case("adamw_bucket150m_master", "adamw", "bucket", 150_000_007, tensors=223, dtype="bf16", limit="over",
              masters=True),
        # the six-view rig's scene, clipped
        _case("adamw_scene2m_clip", "adamw", "scene", 2_000_000, degree=3, limit="over", seen=0.6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "clip", "adamw"))
    kind = rng.choice(("rig", "scene", "scene", "bucket"))
    limit = {"norm": "none", "clip": rng.choice(("over", "over", "in"))}.get(op) or rng.choice(("none", "over", "in"))
    norm = rng.choice(("2", "2", "inf", "1")) if op != "adamw" else "2"
    per = op == "norm" and rng.random() < 0.5
    if kind == "rig":
        return _case(None, op, kind, _log(rng, 1, 4000), norm=norm, per_tensor=per, limit=limit)
    if kind == "scene":
        rows = op == "adamw" and rng.random() < 0.5
        return _case(None, op, kind, _log(rng, 500, 2_000_000), degree=rng.choice((0, 1, 2, 3)), norm=norm,
                     per_tensor=per, limit=limit, seen=round(rng.uniform(0.05, 1.0), 3), row_mask=rows)
    half = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    return _case(None, op, kind, _log(rng, 40_000, 110_000_000), tensors=_log(rng, 3, 400), dtype=half, norm=norm,
                 per_tensor=per, limit=limit, masters=op == "adamw" and half != "fp32" and rng.random() < 0.7)


def _shapes(case):
    n = case["n"]
    if case["kind"] == "rig":
        return [(n, w) for w in RIG_WIDTHS]
    if case["kind"] == "scene":
        return [(n, 3), (n, 4), (n, 3), (n,), (n, (case["degree"] + 1) ** 2, 3)]
    # ragged: sizes spread over four decades, the rest in the last tensor
    r = random.Random(case["tensors"])
    weights = [math.exp(r.uniform(0.0, 9.0)) for _ in range(case["tensors"])]
    sizes = [max(1, int(n * w / sum(weights))) for w in weights[:-1]]
    return [(s,) for s in sizes] + [(n - sum(sizes),)]


def _numel(shape):
    return math.prod(shape)


def _views(flat, shapes):
    at = 0
    out = []
    for s in shapes:
        out.append(flat[at:at + _numel(s)].view(s))
        at += _numel(s)
    return out


def _inputs(case, seed):
    """Tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shapes, dtype = _shapes(case), DTYPES[case["dtype"]]
    total = sum(_numel(s) for s in shapes)

    def rand(n):
        return torch.rand(n, device="cuda", generator=g)

    def randn(n):
        return torch.randn(n, device="cuda", generator=g)

    bucket = case["kind"] == "bucket"
    s = {"case": case, "shapes": shapes, "bucket": bucket}
    grad = randn(total).mul_(torch.exp(randn(total))).mul_(1e-3)
    if case["kind"] == "scene":
        seen = rand(case["n"]) < case["seen"]
        for v in _views(grad, shapes):
            v[~seen] = 0
        s["row_mask"] = seen if case["row_mask"] else None
    else:
        s["row_mask"] = None
    size = float(torch.linalg.vector_norm(grad, float(case["norm"]), dtype=torch.float64))
    s["limit"] = {"none": None, "over": 0.25 * size, "in": 4.0 * size}[case["limit"]]

    def tensors(flat):
        return flat, (_views(flat, shapes) if bucket else [v.clone() for v in _views(flat, shapes)])

    s["flat_grad"], s["grads"] = tensors(grad.to(dtype))
    if case["op"] == "adamw":
        param = randn(total)
        s["flat_master"], s["masters"] = tensors(param) if case["masters"] else (None, None)
        s["flat_param"], s["params"] = tensors(param.to(dtype).clone())
        s["flat_m"], s["ms"] = tensors(randn(total).mul_(3e-4))
        s["flat_v"], s["vs"] = tensors(rand(total).add_(0.05).mul_(2e-6))
        scene = case["kind"] == "scene"
        s["lr"] = list(SCENE_LR) if scene else [1e-3] * len(shapes)
        s["eps"] = 1e-15 if scene else 1e-8
        s["decay"] = 0.0 if scene else 0.01
        # updates taken, and a word that is zero between calls
        s["step"] = torch.tensor([START, 0], dtype=torch.int64, device="cuda")
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------- plain forms --
def _sizes_of(grads, p):
    if p == "inf":
        each = torch.stack([g.float().abs().max() for g in grads])
        return each.max(), each
    if p == "1":
        each = torch.stack([g.float().abs().sum() for g in grads])
        return each.sum(), each
    squares = torch.stack([g.float().square().sum() for g in grads])
    return squares.sum().sqrt(), squares.sqrt()


def _coefficient(total, limit):
    return torch.clamp(limit / (total + CLIP_EPS), max=1.0)


def _plain_update(s, k, coef, c1, c2):
    g, m, v = s["grads"][k].float(), s["ms"][k], s["vs"][k]
    if coef is not None:
        g = g * coef
    w = s["masters"][k] if s["masters"] else s["params"][k].float()
    m1 = BETAS[0] * m + (1.0 - BETAS[0]) * g
    v1 = BETAS[1] * v + (1.0 - BETAS[1]) * g * g
    lr = s["lr"][k]
    w1 = w * (1.0 - lr * s["decay"]) - lr * (m1 / c1) / ((v1 / c2).sqrt() + s["eps"])
    if s["row_mask"] is not None:
        keep = s["row_mask"].view([-1] + [1] * (g.dim() - 1))
        m1, v1, w1 = torch.where(keep, m1, m), torch.where(keep, v1, v), torch.where(keep, w1, w)
    m.copy_(m1)
    v.copy_(v1)
    s["params"][k].copy_(w1)
    if s["masters"]:
        s["masters"][k].copy_(w1)


def _plain(s):
    case = s["case"]
    total = each = None
    if case["op"] != "adamw" or s["limit"] is not None:
        total, each = _sizes_of(s["grads"], case["norm"])
    if case["op"] == "norm":
        return total, each
    coef = None if s["limit"] is None else _coefficient(total, s["limit"])
    if case["op"] == "clip":
        [g.copy_(g.float() * coef) for g in s["grads"]]
        return total, None
    t = (s["step"][0] + 1).float()
    c1, c2 = (-torch.expm1(t * math.log(b)) for b in BETAS)
    [_plain_update(s, k, coef, c1, c2) for k in range(len(s["grads"]))]
    s["step"][0] += 1
    return total, None


def _own(s):
    import xsimgs_b200 as X

    case = s["case"]
    p = float(case["norm"])
    if case["op"] == "norm":
        r = X.gradient_norm(s["grads"], p, per_tensor=case["per_tensor"])
        return r if case["per_tensor"] else (r, None)
    if case["op"] == "clip":
        return X.clip_gradients_(s["grads"], s["limit"], p), None
    total = X.adamw_update_(s["params"], s["grads"], s["ms"], s["vs"], s["step"], lr=s["lr"], betas=BETAS,
                            eps=s["eps"], weight_decay=s["decay"], max_norm=s["limit"], masters=s["masters"],
                            row_mask=s["row_mask"])
    return total, None


def _answer(s, total, each):
    """The outputs of a pass, whole; a bucket's tensors as their flat buffer."""
    case, out = s["case"], {}
    pick = (lambda flat, views: s[flat]) if s["bucket"] else (lambda flat, views: s[views])
    if total is not None:
        out["norm"] = total
    if case["per_tensor"]:
        out["each"] = each
    if case["op"] == "clip":
        out["grads"] = pick("flat_grad", "grads")
    if case["op"] == "adamw":
        out.update(params=pick("flat_param", "params"), m=pick("flat_m", "ms"), v=pick("flat_v", "vs"),
                   step=s["step"])
        if case["masters"]:
            out["masters"] = pick("flat_master", "masters")
    return out


def run(state):
    total, each = (_own if own else _plain)(state)
    out = _answer(state, total, each)
    if state["case"]["op"] == "clip" and state["case"]["limit"] == "over":
        # the limit sinks a little from pass to pass (as an annealed limit does), so that gradients that an
        # earlier pass has scaled down are over it again
        state["limit"] *= 0.9999
    return out


def exact(case, seed):
    """From the definitions, in 64 bits and on the flat tensors of all leaves."""
    s = _inputs(case, seed)
    p = math.inf if case["norm"] == "inf" else int(case["norm"])
    wide = [g.double() for g in s["grads"]]
    each = torch.stack([torch.linalg.vector_norm(g, p) for g in wide])
    total = torch.linalg.vector_norm(each, p)
    factor = 1.0
    if s["limit"] is not None:
        factor = min(1.0, s["limit"] / (float(total) + CLIP_EPS))

    def whole(parts):
        return torch.cat([x.reshape(-1) for x in parts]) if s["bucket"] else parts

    out = {}
    if case["op"] != "adamw" or s["limit"] is not None:
        out["norm"] = total
    if case["per_tensor"]:
        out["each"] = each
    if case["op"] == "clip":
        out["grads"] = whole([g * factor for g in wide])
    if case["op"] == "adamw":
        t = START + 1
        new = {"params": [], "m": [], "v": []}
        for k, g in enumerate(wide):
            w0, m0, v0 = (x[k].double() for x in (s["masters"] or s["params"], s["ms"], s["vs"]))
            g = g * factor
            m = m0 + (g - m0) * (1 - BETAS[0])
            v = v0 + (g ** 2 - v0) * (1 - BETAS[1])
            m_hat, v_hat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
            w = w0 - s["lr"][k] * s["decay"] * w0 - s["lr"][k] * m_hat / (v_hat ** 0.5 + s["eps"])
            if s["row_mask"] is not None:
                gone = ~s["row_mask"]
                w[gone], m[gone], v[gone] = w0[gone], m0[gone], v0[gone]
            for name, x in (("params", w), ("m", m), ("v", v)):
                new[name].append(x)
        out.update({name: whole(x) for name, x in new.items()}, step=None)
        if case["masters"]:
            out["masters"] = out["params"]
    return out


def work(case):
    """Bytes that no form can do without: each input read once, each output written once."""
    sizes = [_numel(s) for s in _shapes(case)]
    total, size = sum(sizes), BYTES[case["dtype"]]
    read = total * size
    if case["op"] == "norm":
        return {"bytes": read, "flops": 2 * total}
    if case["op"] == "clip":
        over = case["limit"] == "over"
        return {"bytes": read * (2 if over else 1), "flops": (3 if over else 2) * total}
    # rows that are not seen need no update; their gradients are still read where there is a norm
    share = case["seen"] if case["row_mask"] else 1.0
    moved = 16 + size + (8 + size if case["masters"] else 2 * size)
    grads_only = 0 if case["limit"] == "none" else (1.0 - share) * size
    mask = case["n"] if case["row_mask"] else 0
    return {"bytes": int(total * (share * moved + grads_only)) + mask, "flops": int(total * share * 14)}
