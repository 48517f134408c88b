"""CPU checks of the gradient norm, clipping and AdamW entries: refusals that
happen before any CUDA call, through the extension and the C ABI."""
import ctypes as C
import inspect

import pytest
import torch


class Span(C.Structure):
    _fields_ = [("data", C.c_void_p), ("n", C.c_int64), ("dtype", C.c_int32)]


class AdamSpan(C.Structure):
    _fields_ = [(k, C.c_void_p) for k in ("param", "grad", "exp_avg", "exp_avg_sq", "master", "row_mask")] + \
               [("n", C.c_int64), ("row_size", C.c_int64), ("param_dtype", C.c_int32), ("grad_dtype", C.c_int32)] + \
               [(k, C.c_double) for k in ("lr", "beta1", "beta2", "eps", "weight_decay")]


@pytest.fixture(scope="module")
def lib():
    from xsimgs_b200 import capi
    lib = capi.lib()
    lib.xsg_grad_norm_workspace_size.restype = C.c_size_t
    lib.xsg_grad_norm_workspace_size.argtypes = [C.c_int64]
    return lib


def test_workspace_size(lib):
    size = lib.xsg_grad_norm_workspace_size
    assert size(0) == 0 and size(-3) == 0
    assert 0 < size(1) <= size(1000) <= size(5000) < 1 << 20
    lib.xsg_grad_norm_workspace_bytes.restype = lib.xsg_adamw_workspace_bytes.restype = C.c_size_t
    for n, need in ((8, 0), (1 << 22, size(1))):
        assert lib.xsg_grad_norm_workspace_bytes((Span * 1)(Span(None, n, 0)), C.c_int64(1)) == need
        assert lib.xsg_adamw_workspace_bytes((AdamSpan * 1)(AdamSpan(n=n)), C.c_int64(1)) == need
    many = (Span * 40)(*[Span(None, 1, 0)] * 40)
    assert lib.xsg_grad_norm_workspace_bytes(many, C.c_int64(40)) == size(40)
    assert lib.xsg_grad_norm_workspace_bytes(None, C.c_int64(40)) == 0


def refuse(lib, rc, code, text):
    assert rc == code and text in lib.xsg_last_error(), (rc, lib.xsg_last_error())


def test_c_abi_refusals(lib):
    fake = 1 << 20  # never read: every call below is refused before a launch
    one = (Span * 1)(Span(fake, 8, 0))

    def norm(spans=one, n=1, p=2, out=fake, ws=fake, size=1 << 20):
        return lib.xsg_grad_norm(spans, C.c_int64(n), p, C.c_void_p(out), None, C.c_void_p(ws), C.c_size_t(size), None)

    refuse(lib, norm(n=0), 1, b"at least one tensor")
    refuse(lib, norm(spans=None), 1, b"at least one tensor")
    refuse(lib, norm(out=None), 1, b"null output")
    refuse(lib, norm(p=3), 1, b"norm type")
    large = (Span * 1)(Span(fake, 1 << 22, 0))  # small ones go in one launch, without scratch
    refuse(lib, norm(spans=large, ws=None), 4, b"workspace")
    refuse(lib, norm(spans=large, size=8), 4, b"workspace")
    refuse(lib, norm(spans=(Span * 1)(Span(fake, -1, 0))), 1, b"element count")
    refuse(lib, norm(spans=(Span * 1)(Span(fake, 1 << 40, 0))), 1, b"element count")
    refuse(lib, norm(spans=(Span * 1)(Span(None, 4, 0))), 1, b"null pointer")
    refuse(lib, norm(spans=(Span * 1)(Span(fake + 2, 4, 0))), 1, b"misaligned")
    refuse(lib, norm(spans=(Span * 1)(Span(fake, 4, 7))), 1, b"element type")

    def clip(limit):
        return lib.xsg_clip_grads(one, C.c_int64(1), 2, C.c_float(limit), C.c_void_p(fake), C.c_void_p(fake),
                                  C.c_size_t(1 << 20), None)

    for bad in (-1.0, float("inf"), float("nan")):
        refuse(lib, clip(bad), 1, b"max_norm")

    def adamw(step=fake, ws=fake, max_norm=-1.0, **kw):
        f = dict(param=fake, grad=fake, exp_avg=fake, exp_avg_sq=fake, n=8, lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8)
        f.update(kw)
        s = (AdamSpan * 1)(AdamSpan(**f))
        return lib.xsg_adamw_update(s, C.c_int64(1), C.c_void_p(step), C.c_float(max_norm), 0, None, C.c_void_p(ws),
                                    C.c_size_t(1 << 20 if ws else 0), None)

    refuse(lib, adamw(step=None), 1, b"step counter")
    refuse(lib, adamw(param=None), 1, b"null pointer")
    refuse(lib, adamw(grad=fake + 1), 1, b"misaligned")
    refuse(lib, adamw(exp_avg=fake + 2), 1, b"misaligned")
    refuse(lib, adamw(param_dtype=5), 1, b"element type")
    refuse(lib, adamw(n=-2), 1, b"element count")
    refuse(lib, adamw(row_mask=fake), 1, b"row size")
    refuse(lib, adamw(beta1=1.0), 1, b"betas")
    refuse(lib, adamw(beta2=-0.1), 1, b"betas")
    refuse(lib, adamw(eps=-1.0), 1, b"eps")
    refuse(lib, adamw(lr=float("nan")), 1, b"learning rate")
    refuse(lib, adamw(max_norm=float("inf")), 1, b"max_norm")
    refuse(lib, adamw(n=1 << 22, max_norm=1.0, ws=None), 4, b"workspace")


def test_extension_refusals_without_gpu():
    import xsimgs_b200 as X
    t = torch.zeros(4)
    step = X.adamw_step_counter("cpu", 3)
    assert step.tolist() == [3, 0]
    for call, match in [
        (lambda: X.gradient_norm([]), "at least one"),
        (lambda: X.gradient_norm([t]), "CUDA"),
        (lambda: X.clip_gradients_([], 1.0), "at least one"),
        (lambda: X.clip_gradients_([t], 1.0), "CUDA"),
        (lambda: X.clip_gradients_([t], -1.0), "max_norm"),
        (lambda: X.gradient_norm([t], norm_type=0.5), "norm_type"),
        (lambda: X.adamw_update_([], [], [], [], step, lr=0.1), "at least one"),
        (lambda: X.adamw_update_([t], [t], [t], [t], step, lr=0.1), "CUDA"),
        (lambda: X.adamw_update_([t], [], [t], [t], step, lr=0.1), "same length"),
        (lambda: X.adamw_update_([t], [t], [t], [t], step, lr=[0.1, 0.2, 0.3]), "one value"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()
    for call in (lambda: X.gradient_norm([1.0]), lambda: X.gradient_norm(3), lambda: X.clip_gradients_([None], 1.0),
                 lambda: X.adamw_update_([t], [t], [t], [t], step, lr="fast")):
        with pytest.raises(TypeError):
            call()


def test_optimizer_arguments():
    import xsimgs_b200 as X
    p = torch.zeros(3, requires_grad=True)
    for bad in (dict(lr=-1.0), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(betas=(0.9, 1.0))):
        with pytest.raises(ValueError):
            X.AdamW([p], **bad)
    opt = X.AdamW([dict(params=[p], lr=0.5)], lr=0.1, betas=(0.8, 0.9))
    assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["betas"] == (0.8, 0.9)
    assert opt.step() is None  # no gradients: nothing to do
    assert "row_masks" in inspect.signature(opt.step).parameters


def test_row_masks_cover_whole_rows(lib):
    # a mask holds n / row_size bytes: elements past the last whole row would be looked up behind it
    fake = 1 << 20

    def adamw(n, row_size):
        s = (AdamSpan * 1)(AdamSpan(param=fake, grad=fake, exp_avg=fake, exp_avg_sq=fake, row_mask=fake, n=n,
                                    row_size=row_size, lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8))
        return lib.xsg_adamw_update(s, C.c_int64(1), C.c_void_p(fake), C.c_float(-1.0), 0, None, None, C.c_size_t(0),
                                    None)

    for n, row_size in ((10, 4), (3, 4), (1, 1 << 20), (1 << 20, 3)):
        refuse(lib, adamw(n, row_size), 1, b"multiple of the row size")


def test_words_of_a_call_are_aligned(lib):
    # norms, the step counter and the scratch's 64-bit sums: an address between words is refused, not launched with
    fake, size = 1 << 20, 1 << 20
    spans = (Span * 1)(Span(fake, 1 << 22, 0))

    def norm(out=fake, norms=None, ws=fake):
        return lib.xsg_grad_norm(spans, C.c_int64(1), 2, C.c_void_p(out), C.c_void_p(norms), C.c_void_p(ws),
                                 C.c_size_t(size), None)

    def clip(out=fake, ws=fake):
        return lib.xsg_clip_grads(spans, C.c_int64(1), 2, C.c_float(1.0), C.c_void_p(out), C.c_void_p(ws),
                                  C.c_size_t(size), None)

    def adamw(step=fake, out=fake, ws=fake, n=1 << 22):
        s = (AdamSpan * 1)(AdamSpan(param=fake, grad=fake, exp_avg=fake, exp_avg_sq=fake, n=n, lr=0.1, beta1=0.9,
                                    beta2=0.99, eps=1e-8))
        return lib.xsg_adamw_update(s, C.c_int64(1), C.c_void_p(step), C.c_float(1.0), 0, C.c_void_p(out),
                                    C.c_void_p(ws), C.c_size_t(size), None)

    for rc in (lambda: norm(out=fake + 2), lambda: norm(norms=fake + 1), lambda: norm(ws=fake + 4),
               lambda: clip(out=fake + 1), lambda: clip(ws=fake + 1), lambda: adamw(step=fake + 4),
               lambda: adamw(out=fake + 3), lambda: adamw(ws=fake + 2), lambda: adamw(step=fake + 1, n=8)):
        refuse(lib, rc(), 1, b"misaligned")


def stock_checkpoint(updates=50, dtype=torch.float32):
    # what torch.optim.AdamW leaves behind: an update count with each parameter, none for all
    torch.manual_seed(1)
    ps = [torch.randn(7, 3, dtype=dtype, requires_grad=True), torch.randn(5, dtype=dtype, requires_grad=True)]
    opt = torch.optim.AdamW(ps, lr=1e-2)
    for _ in range(updates):
        for p in ps:
            p.grad = torch.randn_like(p)
        opt.step()
    return ps, opt.state_dict()


def test_optimizer_takes_the_count_of_a_stock_checkpoint():
    import xsimgs_b200 as X
    ps, saved = stock_checkpoint()
    opt = X.AdamW(ps)
    opt.load_state_dict(saved)
    assert opt._step.tolist() == [50, 0]
    for i, p in enumerate(ps):
        assert set(opt.state[p]) == {"exp_avg", "exp_avg_sq"}
        for k in opt.state[p]:
            assert torch.equal(opt.state[p][k], saved["state"][i][k])
    again = opt.state_dict()
    assert again["updates"] == 50
    # the count survives what keeps state and groups alone, as sharded and converted checkpoints do
    other = X.AdamW(ps)
    other.load_state_dict({k: again[k] for k in ("state", "param_groups")})
    assert other._step.tolist() == [50, 0]
    fresh = X.AdamW(ps)
    fresh.load_state_dict({k: v for k, v in X.AdamW(ps).state_dict().items() if k != "updates"})
    assert fresh._step.tolist() == [0, 0]


def test_optimizer_refuses_moments_without_one_count():
    import xsimgs_b200 as X
    ps, saved = stock_checkpoint(3)
    differ = {**saved, "state": {i: {**s, "step": s["step"] + i} for i, s in saved["state"].items()}}
    missing = {**saved, "state": {i: {k: v for k, v in s.items() if k != "step" or i} for i, s in
                                  saved["state"].items()}}
    for bad in (differ, missing):
        opt = X.AdamW(ps, lr=0.25)
        with pytest.raises(ValueError, match="updates"):
            opt.load_state_dict(bad)
        assert not opt.state and opt._step is None and opt.param_groups[0]["lr"] == 0.25  # as it was


def test_optimizer_completes_a_loaded_state():
    # moments of 32-bit or stock training on half-precision parameters: the missing master comes from the parameter
    import xsimgs_b200 as X
    ps, saved = stock_checkpoint(3, torch.bfloat16)
    opt = X.AdamW(ps)
    opt.load_state_dict(saved)
    for i, p in enumerate(ps):
        s = opt._state(p)
        assert s["master"].dtype == torch.float32 and torch.equal(s["master"], p.detach().float())
        assert torch.equal(s["exp_avg"], saved["state"][i]["exp_avg"].float())
        kept = s["master"]
        assert opt._state(p)["master"] is kept
    p = torch.zeros(3, requires_grad=True)
    opt = X.AdamW([p])
    opt.state[p]["exp_avg"] = torch.ones(3)
    s = opt._state(p)
    assert torch.equal(s["exp_avg"], torch.ones(3)) and torch.equal(s["exp_avg_sq"], torch.zeros(3)) and len(s) == 2


def test_optimizer_refuses_checkpoints_of_other_rules():
    import xsimgs_b200 as X
    ps, _ = stock_checkpoint(1)
    for cls, kw, match in ((torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
                           (torch.optim.AdamW, dict(maximize=True), "maximize"),
                           (torch.optim.Adam, dict(weight_decay=0.1), "decay")):
        stock = cls(ps, **kw)
        stock.step()
        opt = X.AdamW(ps)
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(stock.state_dict())
        assert not opt.state and opt._step is None
    stock = torch.optim.Adam(ps)  # without decay the rules are the same
    stock.step()
    opt = X.AdamW(ps)
    opt.load_state_dict(stock.state_dict())
    assert opt._step.tolist() == [1, 0]


def test_optimizer_step_returns_the_closure_s_loss():
    import xsimgs_b200 as X
    p = torch.zeros(3, requires_grad=True)
    opt = X.AdamW([p], max_norm=1.0)
    assert opt.step(lambda: 2.5) == 2.5 and opt.grad_norm is None  # no gradients: no update, no norm
    assert opt.step() is None


def test_options_fit_32_bits(lib):
    # finite in 64 bits, infinite in the 32 of the update: inf * 0 would make NaN of untouched parameters
    fake = 1 << 20
    for kw in (dict(lr=1e39), dict(lr=-1e39), dict(lr=1e20, weight_decay=1e20), dict(lr=1e-3, weight_decay=1e308)):
        f = dict(param=fake, grad=fake, exp_avg=fake, exp_avg_sq=fake, n=8, beta1=0.9, beta2=0.99, eps=1e-8)
        s = (AdamSpan * 1)(AdamSpan(**{**f, **kw}))
        refuse(lib, lib.xsg_adamw_update(s, C.c_int64(1), C.c_void_p(fake), C.c_float(-1.0), 0, None, None,
                                         C.c_size_t(0), None), 1, b"learning rate")
