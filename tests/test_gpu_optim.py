"""Gradient norm, clipping and AdamW update (csrc/optim.cu) against the
definitions in 64 bits.

Tolerances, with u = 2^-24 (half an ulp of 32 bits):
  norm    a sum of non-negative terms in which at most 16 terms meet in 32
          bits before they go on in 64: relative error of the sum <= 17 u, of
          its root <= 9 u, one rounding to 32 bits: 10 u;
  factor  the norm's error, the rounding of norm + 1e-6 and of the quotient:
          12 u; a scaled 32-bit entry one rounding more: 13 u.  A 16-bit entry
          is off by half an ulp of its type and that 13 u;
  AdamW   m and v: each product and sum rounds once, the gradient carries the
          factor's 12 u (twice in v): 16 u and 32 u of the sum of the
          absolute terms.  w: two roundings of w itself, and the update's
          relative error: m's 16 u, half of v's 32 u, the two bias
          corrections (4 u each), quotient, root, products (6 u): below 48 u
          of lr |m|' / denominator, |m|' with absolute terms.
"""
import math

import pytest
import torch

import xsimgs_b200 as X

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
CLIP_EPS = 1e-6


def norm64(ts, p):
    flat = torch.cat([t.detach().double().reshape(-1).cpu() for t in ts]) if ts else torch.zeros(0).double()
    if flat.numel() == 0:
        return 0.0
    return float(flat.abs().max() if p == math.inf else flat.abs().pow(p).sum() ** (1.0 / p))


def make(sizes, dtype, seed=0, device="cuda", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtype).to(device) for s in sizes]


SIZE_SETS = {
    "one": [1],
    "empty": [0, 0],
    "some_empty": [0, 5, 0, 0, 7, 0],
    "vector_edges": [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33],
    "tile_edges": [2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193],
    "leaves": [3 * 1001, 4 * 1001, 3 * 1001, 1001, 48 * 1001],
    "long": [3_000_001, 5],
    "many": [(7 * i) % 41 for i in range(1500)],
}


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", SIZE_SETS)
def test_norm(name, dtype, p):
    ts = make(SIZE_SETS[name], dtype, seed=len(name))
    total, each = X.gradient_norm(ts, p, per_tensor=True)
    assert total.shape == () and total.dtype == torch.float32 and each.shape == (len(ts),)
    alone = X.gradient_norm(ts, p)
    assert torch.equal(alone, total)
    want = norm64(ts, p)
    assert abs(float(total) - want) <= 10 * U * want
    for got, t in zip(each.tolist(), ts):
        w = norm64([t], p)
        assert abs(got - w) <= 10 * U * w


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_norm_mixed_types_offsets_and_layouts(p):
    base = make([5000], torch.float32, 1)[0]
    half = make([5000], torch.bfloat16, 2)[0]
    f16 = make([5000], torch.float16, 3)[0]
    m = make([60 * 70], torch.float32, 4)[0].view(60, 70)
    ts = [base[1:4097], half[3:], f16[5:11], m.t(), m[:, 3:9], base[:1].expand(300), half[7:8], base[::3],
          make([4 * 5 * 6], torch.float32, 5)[0].view(4, 5, 6).permute(2, 0, 1), base[4990:4990]]
    total, each = X.gradient_norm(ts, p, per_tensor=True)
    assert abs(float(total) - norm64(ts, p)) <= 10 * U * norm64(ts, p)
    for got, t in zip(each.tolist(), ts):
        assert abs(got - norm64([t], p)) <= 10 * U * norm64([t], p)


@pytest.mark.parametrize("value", [1e30, 1e-30, 1e-42, 3e38])
@pytest.mark.parametrize("p", [2.0, math.inf])
def test_norm_neither_overflows_nor_vanishes(value, p):
    t = torch.full((777,), value, device="cuda")
    t[::2] *= -0.5
    want = norm64([t], p)
    got = float(X.gradient_norm([t, torch.zeros(5000, device="cuda")], p))
    if want > torch.finfo(torch.float32).max:
        assert got == math.inf
    else:
        assert abs(got - want) <= 10 * U * want + TINY[torch.float32]


def test_norm_mixes_magnitudes():
    for dtype in (torch.float32, torch.bfloat16):
        t = torch.zeros(100_003, device="cuda", dtype=dtype)
        t[7], t[40_000], t[99_999] = 3e25, 4e25, 1e-20
        want = norm64([t], 2)
        assert abs(float(X.gradient_norm([t])) - want) <= 10 * U * want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("at", [0, 4100, 9998])
def test_norm_shows_nan_and_inf(dtype, p, at):
    for bad, test in ((math.nan, math.isnan), (math.inf, lambda x: x == math.inf), (-math.inf, lambda x: x == math.inf)):
        ts = make([9999, 3], dtype, 1)
        ts[0][at] = bad
        total, each = X.gradient_norm(ts, p, per_tensor=True)
        assert test(float(total)) and test(float(each[0])) and math.isfinite(float(each[1]))
    ts[0][at], ts[0][17] = math.nan, math.inf
    assert math.isnan(float(X.gradient_norm(ts, p)))


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", SIZE_SETS)
def test_clip(name, dtype, p):
    ts = make(SIZE_SETS[name], dtype, seed=3)
    before = [t.double().cpu() for t in ts]
    norm = norm64(ts, p)
    limit = 0.3 * norm if norm else 1.0
    got = X.clip_gradients_(ts, limit, p)
    assert abs(float(got) - norm) <= 10 * U * norm
    c = min(1.0, limit / (norm + CLIP_EPS))
    for t, b in zip(ts, before):
        want = b * c
        off = (t.double().cpu() - want).abs()
        assert (off <= (HALF_ULP[dtype] + 13 * U) * want.abs() + TINY[dtype]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_within_the_limit_changes_nothing(dtype):
    ts = make([4097, 3, 0, 129], dtype)
    before = [t.clone() for t in ts]
    versions = [t._version for t in ts]
    norm = norm64(ts, 2)
    assert abs(float(X.clip_gradients_(ts, 2 * norm)) - norm) <= 10 * U * norm
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    assert all(t._version > v for t, v in zip(ts, versions))


def test_clip_offsets_and_orders():
    flat = make([70_000], torch.float32, 5)[0]
    half = make([70_000], torch.bfloat16, 6)[0]
    ts = [flat[1:30_002], flat[30_002:30_005], half[3:50_000], half[50_000:50_001], flat[40_000:46_000].view(60, 100).t()]
    keep_f, keep_h = flat.clone(), half.clone()
    norm = norm64(ts, 2)
    X.clip_gradients_(ts, 0.1 * norm)
    c = 0.1 * norm / (norm + CLIP_EPS)
    touched = torch.zeros(70_000, dtype=torch.bool, device="cuda")
    touched[1:30_005] = True
    touched[40_000:46_000] = True
    assert torch.equal(flat[~touched], keep_f[~touched])
    assert ((flat - keep_f * c).abs()[touched] <= 16 * U * keep_f.abs()[touched]).all()
    assert torch.equal(half[:3], keep_h[:3]) and torch.equal(half[50_001:], keep_h[50_001:])
    assert ((half.float() - keep_h.float() * c).abs()[3:50_001] <=
            (HALF_ULP[torch.bfloat16] + 16 * U) * keep_h.float().abs()[3:50_001]).all()


def test_clip_limit_zero_and_nonfinite():
    ts = make([5000], torch.float32)
    X.clip_gradients_(ts, 0.0)
    assert (ts[0] == 0).all()
    ts = make([5000], torch.float32)
    ts[0][9] = math.inf
    assert float(X.clip_gradients_(ts, 1.0)) == math.inf
    assert math.isnan(float(ts[0][9])) and (ts[0][10:] == 0).all()
    ts = make([5000], torch.float32)
    ts[0][9] = math.nan
    X.clip_gradients_(ts, 1.0)
    assert torch.isnan(ts[0]).all()


# ----------------------------------------------------------------- AdamW --
def adamw64(w, g, m, v, t, lr, betas, eps, decay, c=1.0):
    """New w, m, v in 64 bits and the bounds of their 32-bit errors."""
    w, g, m, v = (x.double().cpu() for x in (w, g, m, v))
    g = g * c
    b1, b2 = betas
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    m_abs = b1 * m.abs() + (1 - b1) * g.abs()
    den = (v1 / (1 - b2 ** t)).sqrt() + eps
    scale = lr / (1 - b1 ** t)
    w1 = w - lr * decay * w - scale * m1 / den
    tiny = 2.0 ** -149
    return (w1, m1, v1), (3 * U * (w.abs() + w1.abs()) + 48 * U * scale * m_abs / den, 16 * U * m_abs + 4 * tiny,
                          32 * U * v1 + 8 * tiny)


def state_for(sizes, dtype, seed, gdtype=None, masters=False):
    w = make(sizes, torch.float32, seed)
    g = make(sizes, gdtype or dtype, seed + 1, scale=1e-3)
    m = make(sizes, torch.float32, seed + 2, scale=3e-4)
    v = [x.square().mul_(1e-6).add_(1e-9) for x in make(sizes, torch.float32, seed + 3)]
    p = [x.to(dtype) for x in w]
    return p, g, m, v, (w if masters else None)


def check_update(p, g, m, v, masters, old, t, lr, betas, eps, decay, c=1.0, masks=None):
    for i in range(len(p)):
        ow, og, om, ov = old[i]
        (w1, m1, v1), (dw, dm, dv) = adamw64(ow, og, om, ov, t, lr[i], betas, eps, decay, c)
        new_w = (masters[i] if masters else p[i]).double().cpu()
        new_m, new_v, new_p = m[i].double().cpu(), v[i].double().cpu(), p[i].double().cpu()
        rows = torch.ones(w1.shape, dtype=torch.bool)
        if masks is not None and masks[i] is not None:
            rows = masks[i].bool().cpu().view([-1] + [1] * (w1.dim() - 1)).expand(w1.shape)
            assert torch.equal(new_m[~rows], om.double().cpu()[~rows])
            assert torch.equal(new_v[~rows], ov.double().cpu()[~rows])
            assert torch.equal(new_w[~rows], ow.double().cpu()[~rows])
        dt = torch.float32 if masters else p[i].dtype
        assert ((new_m - m1).abs() <= dm)[rows].all()
        assert ((new_v - v1).abs() <= dv)[rows].all()
        assert ((new_w - w1).abs() <= dw + HALF_ULP[dt] * w1.abs() * 1.01 + TINY[dt])[rows].all()
        if masters:
            assert torch.equal(p[i][rows.to(p[i].device)], masters[i].to(p[i].dtype)[rows.to(p[i].device)])


@pytest.mark.parametrize("name", SIZE_SETS)
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16", "bf16_master", "f32_bf16grad"])
@pytest.mark.parametrize("clip", [False, True])
def test_adamw(name, kind, clip):
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "bf16_master": torch.bfloat16,
             "f32_bf16grad": torch.float32}[kind]
    p, g, m, v, masters = state_for(SIZE_SETS[name], dtype, 11, torch.bfloat16 if kind == "f32_bf16grad" else None,
                                    kind == "bf16_master")
    lr = [1e-3 * (1 + i % 3) for i in range(len(p))]
    step = X.adamw_step_counter("cuda", 4)
    for t in (5, 6):
        old = [(a.clone(), b.clone(), c.clone(), d.clone()) for a, b, c, d in zip(masters or p, g, m, v)]
        norm = norm64(g, 2)
        limit = 0.2 * norm if norm else 1.0
        got = X.adamw_update_(p, g, m, v, step, lr=lr, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02,
                              max_norm=limit if clip else None, masters=masters)
        assert (got is None) == (not clip)
        if clip:
            assert abs(float(got) - norm) <= 10 * U * norm
        assert all(torch.equal(b, o[1]) for b, o in zip(g, old))
        check_update(p, g, m, v, masters, old, t, lr, (0.9, 0.99), 1e-8, 0.02,
                     min(1.0, limit / (norm + CLIP_EPS)) if clip else 1.0)
        assert step.tolist() == [t, 0]


def test_adamw_first_step_and_zero_gradients():
    # t = 1 from zero moments: the update is lr * sign(g); rows without gradient stay (0 / eps)
    p, g = make([3001], torch.float32, 1), make([3001], torch.float32, 2)
    g[0][::3] = 0
    m, v = [torch.zeros_like(p[0])], [torch.zeros_like(p[0])]
    before = p[0].clone()
    step = X.adamw_step_counter("cuda")
    X.adamw_update_(p, g, m, v, step, lr=0.01, eps=1e-15)
    assert torch.equal(p[0][::3], before[::3])
    d = (before - p[0]).double()
    assert ((d - 0.01 * g[0].sign().double()).abs() <= 3 * U * (before.abs() + 0.01) + 48 * U * 0.01).all()
    assert step.tolist() == [1, 0]


@pytest.mark.parametrize("t", [1, 10, 1000, 100_000, 10_000_000])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.0, 0.0), (0.99, 0.9999)])
def test_adamw_bias_corrections(t, betas):
    p, g, m, v, _ = state_for([513], torch.float32, 21)
    old = [(p[0].clone(), g[0].clone(), m[0].clone(), v[0].clone())]
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", t - 1), lr=0.01, betas=betas, eps=1e-12)
    check_update(p, g, m, v, None, old, t, [0.01], betas, 1e-12, 0.0)


ROW_SHAPES = [(1,), (5,), (4099,), (1, 3), (7, 3), (1000, 3), (1367, 4), (683, 1), (700, 16, 3), (33, 5000), (0, 3)]


@pytest.mark.parametrize("shape", ROW_SHAPES)
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("kind", ["f32", "bf16_master"])
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_rows(shape, share, kind, clip):
    n = math.prod(shape)
    p, g, m, v, masters = state_for([n], torch.bfloat16 if kind == "bf16_master" else torch.float32, 31,
                                    masters=kind == "bf16_master")
    p, g, m, v = ([x[0].view(shape)] for x in (p, g, m, v))
    masters = [masters[0].view(shape)] if masters else None
    mask = torch.rand(shape[0], generator=torch.Generator().manual_seed(5)).lt(share).cuda()
    old = [((masters or p)[0].clone(), g[0].clone(), m[0].clone(), v[0].clone())]
    norm = norm64(g, 2)
    limit = 0.5 * norm if norm else 1.0
    before = p[0].clone()
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 9), lr=0.01, row_mask=mask, masters=masters,
                    max_norm=limit if clip else None)
    check_update(p, g, m, v, masters, old, 10, [0.01], (0.9, 0.999), 1e-8, 0.0,
                 min(1.0, limit / (norm + CLIP_EPS)) if clip else 1.0, [mask])
    assert torch.equal(p[0][~mask], before[~mask])


def test_adamw_rows_one_mask_for_all_leaves_and_masked_nan():
    n = 2051
    shapes = [(n, 3), (n, 4), (n, 3), (n,), (n, 16, 3)]
    flat = state_for([math.prod(s) for s in shapes], torch.float32, 41)
    p, g, m, v = ([x.view(s) for x, s in zip(xs, shapes)] for xs in flat[:4])
    mask = torch.arange(n, device="cuda") % 5 < 2
    for x in g:
        x[~mask] = math.nan
    old = [tuple(x.clone() for x in q) for q in zip(p, g, m, v)]
    lr = [1e-4, 1e-3, 5e-3, 5e-2, 2e-3]
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 9), lr=lr, eps=1e-15, row_mask=mask)
    check_update(p, g, m, v, None, old, 10, lr, (0.9, 0.999), 1e-15, 0.0, 1.0, [mask] * 5)


def test_adamw_mask_list_and_uint8():
    p, g, m, v, _ = state_for([30, 28], torch.float32, 51)
    p[0], g[0], m[0], v[0] = (x[0].view(10, 3) for x in (p, g, m, v))
    mask = (torch.arange(10, device="cuda") % 2 * 255).to(torch.uint8)
    old = [tuple(x.clone() for x in q) for q in zip(p, g, m, v)]
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda"), lr=0.01, row_mask=[mask, None])
    check_update(p, g, m, v, None, old, 1, [0.01, 0.01], (0.9, 0.999), 1e-8, 0.0, 1.0, [mask, None])


@pytest.mark.parametrize("offsets", [(1, 1, 1, 1), (0, 1, 2, 3), (7, 7, 7, 7), (0, 0, 0, 1)])
@pytest.mark.parametrize("kind", ["f32", "bf16_master"])
def test_adamw_offsets(offsets, kind):
    n = 10_007
    p, g, m, v, masters = state_for([n + 16], torch.bfloat16 if kind == "bf16_master" else torch.float32, 61,
                                    masters=kind == "bf16_master")
    whole = [p[0], g[0], m[0], v[0]]
    kept = [x.clone() for x in whole]
    p, g, m, v = ([x[o:o + n]] for x, o in zip(whole, offsets))
    mw = masters[0] if masters else None
    masters = [mw[offsets[0]:offsets[0] + n]] if masters else None
    old = [((masters or p)[0].clone(), g[0].clone(), m[0].clone(), v[0].clone())]
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 2), lr=0.01, masters=masters)
    check_update(p, g, m, v, masters, old, 3, [0.01], (0.9, 0.999), 1e-8, 0.0)
    for x, k, o in zip(whole, kept, offsets):
        assert torch.equal(x[:o], k[:o]) and torch.equal(x[o + n:], k[o + n:])


def test_adamw_orders_of_dimensions():
    p, g, m, v, _ = state_for([60 * 70], torch.float32, 71)
    p, m, v = ([x[0].view(60, 70).t()] for x in (p, m, v))
    for grad in (g[0].view(60, 70).t(), g[0].view(70, 60), g[0][:70].view(70, 1).expand(70, 60)):
        old = [(p[0].clone(), grad.clone(), m[0].clone(), v[0].clone())]
        X.adamw_update_(p, [grad], m, v, X.adamw_step_counter("cuda"), lr=0.01)
        check_update(p, [grad], m, v, None, old, 1, [0.01], (0.9, 0.999), 1e-8, 0.0)


def test_adamw_many_groups_and_tensors():
    n = 700  # more tensors and more distinct learning rates than one launch takes
    p, g, m, v, _ = state_for([1 + i % 5 for i in range(n)], torch.float32, 81)
    lr = [1e-3 * (1 + i % 90) for i in range(n)]
    old = [tuple(x.clone() for x in q) for q in zip(p, g, m, v)]
    step = X.adamw_step_counter("cuda", 2)
    norm = norm64(g, 2)
    X.adamw_update_(p, g, m, v, step, lr=lr, max_norm=0.5 * norm)
    check_update(p, g, m, v, None, old, 3, lr, (0.9, 0.999), 1e-8, 0.0, 0.5 * norm / (norm + CLIP_EPS))
    assert step.tolist() == [3, 0]


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_adamw_skips_nonfinite(bad):
    p, g, m, v, _ = state_for([5000, 3], torch.float32, 91)
    g[0][4999] = bad
    before = [x.clone() for x in p + m + v]
    step = X.adamw_step_counter("cuda", 7)
    norm = X.adamw_update_(p, g, m, v, step, lr=0.01, skip_nonfinite=True)
    assert not math.isfinite(float(norm))
    assert all(torch.equal(a, b) for a, b in zip(p + m + v, before)) and step.tolist() == [7, 0]
    g[0][4999] = 0.5
    X.adamw_update_(p, g, m, v, step, lr=0.01, max_norm=1.0, skip_nonfinite=True)
    assert step.tolist() == [8, 0] and not torch.equal(p[0], before[0])


def test_same_bits_every_run():
    ts = make([1_000_003, 17, 400_000], torch.float32, 3)
    norms = {float(X.gradient_norm(ts)) for _ in range(5)}
    assert len(norms) == 1
    results = []
    for _ in range(2):
        p, g, m, v, _ = state_for([1_000_003, 5], torch.float32, 3)
        step = X.adamw_step_counter("cuda")
        for _ in range(3):
            X.adamw_update_(p, g, m, v, step, lr=0.01, max_norm=0.1)
        results.append(p[0])
    assert torch.equal(*results)


def test_other_stream_and_graph():
    p, g, m, v, _ = state_for([100_000, 7], torch.float32, 5)
    q, h, k, w, _ = state_for([100_000, 7], torch.float32, 5)
    a, b = X.adamw_step_counter("cuda"), X.adamw_step_counter("cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        X.adamw_update_(p, g, m, v, a, lr=0.01, max_norm=0.1)  # warm-up on the capturing stream
        X.clip_gradients_(g, 0.5)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        X.adamw_update_(p, g, m, v, a, lr=0.01, max_norm=0.1)
        X.clip_gradients_(g, 0.05)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    X.adamw_update_(q, h, k, w, b, lr=0.01, max_norm=0.1)
    X.clip_gradients_(h, 0.5)
    for _ in range(3):
        X.adamw_update_(q, h, k, w, b, lr=0.01, max_norm=0.1)
        X.clip_gradients_(h, 0.05)
    assert a.tolist() == b.tolist() == [4, 0]
    assert all(torch.equal(x, y) for x, y in zip(p + g + m + v, q + h + k + w))


def test_past_32_bits():
    n = (1 << 32) + 4097  # elements; 8.6 GB
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[0], t[n - 1], t[1 << 31] = 2.0, 3.0, 6.0
    assert float(X.gradient_norm([t])) == 7.0
    assert float(X.gradient_norm([t], math.inf)) == 6.0
    X.clip_gradients_([t], 3.5)
    assert abs(float(t[n - 1]) - 1.5) < 0.01 and abs(float(t[1 << 31]) - 3.0) < 0.02
    assert int(torch.count_nonzero(t)) == 3


def test_adamw_past_32_bits():
    n = (1 << 31) + 5
    p = torch.zeros((n,), dtype=torch.bfloat16, device="cuda")
    g = torch.zeros((n,), dtype=torch.bfloat16, device="cuda")
    m, v = torch.zeros((n,), device="cuda"), torch.zeros((n,), device="cuda")
    g[n - 1], g[5] = 1.0, -1.0
    X.adamw_update_([p], [g], [m], [v], X.adamw_step_counter("cuda"), lr=0.5)
    assert float(p[n - 1]) == -0.5 and float(p[5]) == 0.5 and int(torch.count_nonzero(p)) == 2
    mask = torch.zeros(n, dtype=torch.bool, device="cuda")
    mask[n - 1] = True
    X.adamw_update_([p], [g], [m], [v], X.adamw_step_counter("cuda", 1), lr=0.5, row_mask=mask)
    assert float(p[n - 1]) == -1.0 and float(p[5]) == 0.5


def test_refusals():
    t = torch.randn(4, 6, device="cuda")
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        X.gradient_norm([t.double()])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        X.gradient_norm([t, torch.zeros(2)])
    with pytest.raises(RuntimeError, match="norm_type"):
        X.gradient_norm([t], 3.0)
    with pytest.raises(RuntimeError, match="dense"):
        X.clip_gradients_([t[:, :3]], 1.0)
    with pytest.raises(RuntimeError, match="dense"):
        X.clip_gradients_([t[:1, :1].expand(3, 3)], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        X.clip_gradients_([t, t], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        X.clip_gradients_([t.view(-1)[:13], t.view(-1)[12:]], 1.0)
    for bad in (math.nan, math.inf, -0.5, 1e39):
        with pytest.raises(RuntimeError, match="max_norm"):
            X.clip_gradients_([t], bad)
    p, g, m, v = (torch.zeros(6, 4, device="cuda") for _ in range(4))
    step = X.adamw_step_counter("cuda")

    def update(p=p, g=g, m=m, v=v, step=step, lr=0.1, **kw):
        return X.adamw_update_([p], [g], [m], [v], step, lr=lr, **kw)

    for kw, match in [
        (dict(p=p.double()), "float32, bfloat16 or float16"), (dict(m=m.half()), "float32"),
        (dict(g=g[:5]), "sizes"), (dict(m=m.t().contiguous().t()), "strides"), (dict(v=p), "shares memory"),
        (dict(g=p), "shares memory"), (dict(p=p.expand(6, 4)[:, :2]), "dense"), (dict(step=torch.zeros(2)), "CUDA"),
        (dict(step=torch.zeros(2, device="cuda")), "int64"), (dict(lr=[0.1, 0.2]), "one value"),
        (dict(lr=math.nan), "learning rate"), (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "eps"),
        (dict(max_norm=math.inf), "max_norm"), (dict(row_mask=torch.ones(5, dtype=torch.bool, device="cuda")), "rows"),
        (dict(row_mask=torch.ones(6, device="cuda")), "bool"), (dict(masters=[p]), "shares memory"),
        (dict(masters=[p, p]), "masters"), (dict(row_mask=[None, None]), "row_mask"),
        (dict(p=torch.zeros((), device="cuda"), g=torch.zeros((), device="cuda"), m=torch.zeros((), device="cuda"),
              v=torch.zeros((), device="cuda"), row_mask=torch.ones(1, dtype=torch.bool, device="cuda")), "rows"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            update(**kw)
    assert step.tolist() == [0, 0]


# ------------------------------------------------------------- optimiser --
def test_optimizer_follows_torch_and_resumes():
    def model(dtype=torch.float32):
        torch.manual_seed(3)
        return [torch.randn(300, 3, device="cuda", dtype=dtype, requires_grad=True),
                torch.randn(41, device="cuda", dtype=dtype, requires_grad=True),
                torch.randn(5, device="cuda", dtype=dtype, requires_grad=True)]

    def groups(ps):
        return [dict(params=ps[:1], lr=1e-2), dict(params=ps[1:], weight_decay=0.1, betas=(0.8, 0.95))]

    a, b = model(), model()
    ours = X.AdamW(groups(a), lr=3e-3, max_norm=0.7)
    theirs = torch.optim.AdamW(groups(b), lr=3e-3, weight_decay=0.0)
    for k in range(6):
        if k == 3:
            saved = ours.state_dict()
            ours = X.AdamW(groups(a), lr=3e-3, max_norm=0.7)
            ours.load_state_dict(saved)
        for ps in (a, b):
            for p in ps:
                p.grad = None
            sum((p * (1 + k) + p.square()).sum() for p in ps[:2]).backward()  # the last has no gradient
        n1 = ours.step()
        n2 = torch.nn.utils.clip_grad_norm_([p for p in b if p.grad is not None], 0.7)
        theirs.step()
        assert abs(float(n1) - float(n2)) <= 1e-5 * float(n2)
        for x, y in zip(a, b):
            assert (x - y).abs().max() <= 1e-6 * (1 + k)


def test_optimizer_masters_survive_a_checkpoint():
    p = torch.randn(1000, device="cuda").to(torch.bfloat16).requires_grad_()
    opt = X.AdamW([p], lr=1e-4)
    p.grad = torch.ones_like(p)
    opt.step()
    first = opt.state[p]["master"].clone()
    again = X.AdamW([p], lr=1e-4)
    again.load_state_dict(opt.state_dict())
    assert again.state[p]["master"].dtype == torch.float32 and torch.equal(again.state[p]["master"], first)
    again.step()
    assert again._step.tolist() == [2, 0]
    assert torch.equal(p, again.state[p]["master"].to(torch.bfloat16))


def test_optimizer_row_masks():
    p = torch.randn(50, 3, device="cuda", requires_grad=True)
    before = p.detach().clone()
    opt = X.AdamW([p], lr=0.1)
    p.grad = torch.ones_like(p)
    mask = torch.arange(50, device="cuda") < 20
    opt.step(row_masks={p: mask})
    assert torch.equal(p.detach()[20:], before[20:]) and (p.detach()[:20] != before[:20]).all()


def test_optimizer_copies_and_pickles():
    import copy
    import pickle
    p = torch.randn(20, 3, device="cuda", requires_grad=True)
    opt = X.AdamW([p], lr=0.1, max_norm=2.0)
    p.grad = torch.ones_like(p)
    opt.step()
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        q = twin.param_groups[0]["params"][0]
        assert twin.max_norm == 2.0 and twin._step.tolist() == [1, 0] and q.data_ptr() != p.data_ptr()
        q.grad = torch.ones_like(q)
        assert float(twin.step()) > 0 and twin._step.tolist() == [2, 0]
    assert opt._step.tolist() == [1, 0]


# ------------------------------------- each form of a call at its limits --
@pytest.mark.parametrize("n", [16_383, 16_384, 16_385, 65_537, 262_143, 262_144, 262_145, 600_011, 1_300_003, 2_700_001])
@pytest.mark.parametrize("tensors", [1, 32, 33])
def test_every_size_of_call(n, tensors):
    # one launch, two launches and each size of tile change over between these
    sizes = [n // (2 * tensors)] * (tensors - 1)
    sizes.append(n - sum(sizes))
    p, g, m, v, _ = state_for(sizes, torch.float32, n % 1000)
    norm = norm64(g, 2)
    total, each = X.gradient_norm(g, per_tensor=True)
    assert torch.equal(total, X.gradient_norm(g))
    assert abs(float(total) - norm) <= 10 * U * norm
    for got, t in zip(each.tolist(), g):
        assert abs(got - norm64([t], 2)) <= 10 * U * norm64([t], 2)
    old = [tuple(x.clone() for x in q) for q in zip(p, g, m, v)]
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 2), lr=0.01, max_norm=0.3 * norm)
    c = 0.3 * norm / (norm + CLIP_EPS)
    check_update(p, g, m, v, None, old, 3, [0.01] * tensors, (0.9, 0.999), 1e-8, 0.0, c)
    before = [t.double() for t in g]
    X.clip_gradients_(g, 0.3 * norm)
    for t, b in zip(g, before):
        assert ((t.double() - b * c).abs() <= 14 * U * (b * c).abs() + TINY[torch.float32]).all()


@pytest.mark.parametrize("count", [1, 100, 2047, 2048, 2049, 5000])
@pytest.mark.parametrize("masked", [False, True])
def test_adamw_one_launch_or_two(count, masked):
    p, g, m, v, _ = state_for([count], torch.float32, 7)
    mask = (torch.arange(count, device="cuda") % 3 == 0) if masked else None
    old = [tuple(x.clone() for x in q) for q in zip(p, g, m, v)]
    norm = norm64(g, 2)
    step = X.adamw_step_counter("cuda", 2)
    got = X.adamw_update_(p, g, m, v, step, lr=0.01, max_norm=0.3 * norm, row_mask=mask)
    assert abs(float(got) - norm) <= 10 * U * norm and step.tolist() == [3, 0]
    check_update(p, g, m, v, None, old, 3, [0.01], (0.9, 0.999), 1e-8, 0.0, 0.3 * norm / (norm + CLIP_EPS),
                 [mask] if masked else None)
    before = p[0].clone()
    g[0][0] = math.nan
    X.adamw_update_(p, g, m, v, step, lr=0.01, skip_nonfinite=True)
    assert step.tolist() == [3, 0] and torch.equal(before, p[0])


def test_small_calls_in_a_graph():
    p, g, m, v, _ = state_for([40, 7], torch.float32, 5)
    step = X.adamw_step_counter("cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        X.adamw_update_(p, g, m, v, step, lr=0.01, max_norm=0.1)
        X.clip_gradients_(g, 1e9)
        X.gradient_norm(g, per_tensor=True)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        X.adamw_update_(p, g, m, v, step, lr=0.01, max_norm=0.1)
        X.clip_gradients_(g, 1e9)
        total, each = X.gradient_norm(g, per_tensor=True)
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert step.tolist() == [5, 0]
    assert abs(float(total) - norm64(g, 2)) <= 10 * U * norm64(g, 2)


def test_large_tensors():
    n = 52_000_003  # large tiles, more than the L2 holds
    g = torch.empty(n + 3, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))[3:]
    want = float(torch.linalg.vector_norm(g, dtype=torch.float64))
    assert abs(float(X.gradient_norm([g])) - want) <= 10 * U * want
    total, each = X.gradient_norm([g[:7], g[7:]], per_tensor=True)
    assert abs(float(total) - want) <= 10 * U * want
    before = g.clone()
    X.clip_gradients_([g], 0.25 * want)
    c = 0.25 * want / (want + CLIP_EPS)
    assert ((g.double() - before.double() * c).abs() <= 14 * U * before.double().abs() * c).all()


@pytest.mark.parametrize("kind", ["f32", "bf16_master"])
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_large(kind, clip):
    # a block for each tile, behind the norm's own launch
    sizes = [11_000_001, 3, 9_000_020]
    p, g, m, v, masters = state_for(sizes, torch.bfloat16 if kind == "bf16_master" else torch.float32, 13,
                                    masters=kind == "bf16_master")
    old = [tuple(x.clone() for x in q) for q in zip(masters or p, g, m, v)]
    norm = norm64(g, 2)
    step = X.adamw_step_counter("cuda", 2)
    got = X.adamw_update_(p, g, m, v, step, lr=0.01, masters=masters, max_norm=0.3 * norm if clip else None)
    check_update(p, g, m, v, masters, old, 3, [0.01] * 3, (0.9, 0.999), 1e-8, 0.0,
                 0.3 * norm / (norm + CLIP_EPS) if clip else 1.0)
    assert step.tolist() == [3, 0] and (not clip or abs(float(got) - norm) <= 10 * U * norm)
    g[0][5_000_000] = math.nan
    before = [x.clone() for x in p]
    X.adamw_update_(p, g, m, v, step, lr=0.01, masters=masters, skip_nonfinite=True)
    assert step.tolist() == [3, 0] and all(torch.equal(a, b) for a, b in zip(p, before))


@pytest.mark.parametrize("m0", [0.0, 1e-45, 1e-41, 1e-3])
@pytest.mark.parametrize("v0", [0.0, 1e-45, 1e-41, 1e-30, 1e-6, 1e38])
@pytest.mark.parametrize("eps", [1e-15, 1e-8, 1e-36])
def test_adamw_subnormal_moments(m0, v0, eps):
    p = make([3001], torch.float32, 1)
    g = [torch.zeros(3001, device="cuda")]
    m, v = [torch.full((3001,), m0, device="cuda")], [torch.full((3001,), v0, device="cuda")]
    old = [(p[0].clone(), g[0].clone(), m[0].clone(), v[0].clone())]
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 99), lr=1e-3, eps=eps)
    (w1, m1, v1), (dw, dm, dv) = adamw64(*old[0], 100, 1e-3, (0.9, 0.999), eps, 0.0)
    assert ((m[0].double().cpu() - m1).abs() <= dm).all() and ((v[0].double().cpu() - v1).abs() <= dv).all()
    # the update from the 32-bit moments that were written: near the bottom their rounding is part of the inputs
    mw, vw = m[0].double().cpu(), v[0].double().cpu()
    scale = 1e-3 / (1 - 0.9 ** 100)
    den = (vw / (1 - 0.999 ** 100)).sqrt() + eps
    want = old[0][0].double().cpu() - scale * mw / den
    bound = 3 * U * (old[0][0].double().cpu().abs() + want.abs()) + 48 * U * scale * mw.abs() / den
    assert ((p[0].double().cpu() - want).abs() <= bound).all()


def test_kinds_of_sequences():
    ts = make([5, 9000], torch.float32)
    want = X.gradient_norm(ts)
    assert torch.equal(X.gradient_norm(tuple(ts)), want) and torch.equal(X.gradient_norm(t for t in ts), want)
    for bad in (ts[0], 3, [ts[0], None]):
        with pytest.raises(TypeError, match="grads"):
            X.gradient_norm(bad)


def test_views_that_negate():
    z = torch.randn(500, dtype=torch.complex64, device="cuda").conj()
    neg = z.imag  # a float view with the sign to be turned
    assert neg.is_neg()
    p, g, m, v, _ = state_for([500], torch.float32, 3)
    g = [neg]
    old = [(p[0].clone(), neg.clone(), m[0].clone(), v[0].clone())]
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda"), lr=0.01)
    check_update(p, g, m, v, None, old, 1, [0.01], (0.9, 0.999), 1e-8, 0.0)
    with pytest.raises(RuntimeError, match="negate|dense"):
        X.clip_gradients_([neg], 1.0)


def test_instrumentation():
    from xsimgs_b200 import capi
    p, g, m, v, _ = state_for([70_000], torch.float32, 3)
    step = X.adamw_step_counter("cuda")
    before = capi.launch_count()
    capi.timing_reset()
    capi.timing_enable(True)
    X.gradient_norm(g)
    X.clip_gradients_(g, 1e-3)
    X.adamw_update_(p, g, m, v, step, lr=0.1, max_norm=1.0)
    capi.timing_enable(False)
    assert capi.launch_count() - before == 1 + 2 + 2
    for name in ("grad_norm", "clip_grads", "adamw_update"):
        ms, count = capi.timing_query(name)
        assert count == 1 and 0 < ms < 100
    capi.timing_reset()


# --------------------------------------------- the counter's second word --
def check_either_count(p, g, m, v, old, counts, lr, eps, c=1.0, masks=None):
    """Every element updated once, with one of the counts' bias corrections."""
    for i in range(len(p)):
        found = torch.zeros(p[i].shape, dtype=torch.bool)
        for t in counts:
            (w1, m1, v1), (dw, dm, dv) = adamw64(*old[i], t, lr, (0.9, 0.999), eps, 0.0, c)
            found |= ((p[i].double().cpu() - w1).abs() <= dw + HALF_ULP[torch.float32] * w1.abs() * 1.01)
            near_m, near_v = (m[i].double().cpu() - m1).abs() <= dm, (v[i].double().cpu() - v1).abs() <= dv
        moved = near_m & near_v & found
        if masks is not None:
            rows = masks[i].cpu().view([-1] + [1] * (p[i].dim() - 1)).expand(p[i].shape)
            same = (p[i] == old[i][0]).cpu() & (m[i] == old[i][2]).cpu() & (v[i] == old[i][3]).cpu()
            moved = torch.where(rows, moved, same)
        assert moved.all()


@pytest.mark.parametrize("word", [1, 3, 700, 1 << 20, -1])
@pytest.mark.parametrize("kind", ["plain", "clip", "rows", "rows_clip"])
@pytest.mark.parametrize("n", [3000, 300_000, 3_000_000])
def test_adamw_updates_everything_whatever_the_second_word(word, kind, n):
    # a counter whose second word was left wrong may cost an update's count, but no element its update
    p, g, m, v, _ = state_for([3 * (n // 4), 3 * (n // 12) + 3], torch.float32, 17)
    mask = None
    if "rows" in kind:
        p, g, m, v = ([x.view(-1, 3) for x in xs] for xs in (p, g, m, v))
        mask = [torch.arange(x.shape[0], device="cuda") % 3 < 2 for x in p]
    old = [tuple(x.clone() for x in q) for q in zip(p, g, m, v)]
    norm = norm64(g, 2)
    limit = 0.3 * norm if "clip" in kind else None
    step = torch.tensor([4, word], dtype=torch.int64, device="cuda")
    X.adamw_update_(p, g, m, v, step, lr=0.01, max_norm=limit, row_mask=mask)
    check_either_count(p, g, m, v, old, (5, 6), 0.01, 1e-8, limit / (norm + CLIP_EPS) if limit else 1.0, mask)
    if "clip" in kind:
        assert int(step[0]) == 5


@pytest.mark.parametrize("kind", ["plain", "clip", "rows"])
def test_adamw_shared_counter_on_two_streams(kind):
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    step = X.adamw_step_counter("cuda", 4)
    calls = []
    for k in range(2):
        p, g, m, v, _ = state_for([3 * 700_001 + 300_000 * k], torch.float32, 23 + k)
        mask = None
        if kind == "rows":
            p, g, m, v = ([x.view(-1, 3) for x in xs] for xs in (p, g, m, v))
            mask = [torch.arange(p[0].shape[0], device="cuda") % 3 < 2]
        norm = norm64(g, 2)
        calls.append((p, g, m, v, mask, 0.3 * norm if kind == "clip" else None,
                      0.3 * norm / (norm + CLIP_EPS) if kind == "clip" else 1.0,
                      [tuple(x.clone() for x in q) for q in zip(p, g, m, v)]))
    torch.cuda.synchronize()
    for s, (p, g, m, v, mask, limit, _, _) in zip(streams, calls):
        with torch.cuda.stream(s):
            X.adamw_update_(p, g, m, v, step, lr=0.01, max_norm=limit, row_mask=mask)
    torch.cuda.synchronize()
    for p, g, m, v, mask, _, c, old in calls:
        check_either_count(p, g, m, v, old, (5, 6, 7), 0.01, 1e-8, c, mask)


# ------------------------------------------- checkpoints of stock optimisers --
def test_optimizer_goes_on_from_a_stock_checkpoint():
    def grads(ps, k):
        for p in ps:
            p.grad = (1 + k) * p.detach().sin()

    torch.manual_seed(5)
    a = [torch.randn(300, 3, device="cuda", requires_grad=True), torch.randn(41, device="cuda", requires_grad=True)]
    theirs = torch.optim.AdamW(a, lr=3e-3, weight_decay=0.1)
    for k in range(4):
        grads(a, k)
        theirs.step()
    b = [p.detach().clone().requires_grad_() for p in a]
    ours = X.AdamW(b)
    ours.load_state_dict(theirs.state_dict())
    for k in range(4):
        for ps, opt in ((a, theirs), (b, ours)):
            grads(ps, k)
            opt.step()
        for x, y in zip(a, b):
            assert (x - y).abs().max() <= 1e-6 * (1 + k)
    assert ours._step.tolist() == [8, 0]


def test_optimizer_gives_loaded_half_parameters_masters():
    p = torch.randn(1000, device="cuda").to(torch.bfloat16).requires_grad_()
    stock = torch.optim.AdamW([p], lr=1e-3)
    p.grad = torch.ones_like(p)
    stock.step()
    ours = X.AdamW([p])
    ours.load_state_dict(stock.state_dict())
    before = p.detach().float()
    for k in range(40):  # steps of 1e-5, below the parameter's spacing for most: only masters keep them
        for g in ours.param_groups:
            g["lr"], g["weight_decay"] = 1e-5, 0.0
        ours.step()
    master = ours.state[p]["master"]
    assert torch.equal(p.detach(), master.to(torch.bfloat16)) and ours._step.tolist() == [41, 0]
    assert ((before - master) > 3e-4).all()  # 40 steps of 1e-5 against gradients of one


def test_optimizer_closure():
    p = torch.full((300,), 2.0, device="cuda", requires_grad=True)
    q = p.detach().clone().requires_grad_()
    opt, other = X.AdamW([p], lr=0.1, max_norm=1.0), X.AdamW([q], lr=0.1, max_norm=1.0)

    def closure():
        opt.zero_grad()
        loss = p.square().sum()
        loss.backward()
        return loss

    loss = opt.step(closure)
    assert float(loss) == 1200.0
    q.grad = 2.0 * q.detach()
    norm = other.step()
    assert torch.equal(opt.grad_norm, norm) and other.grad_norm is norm
    assert torch.equal(p, q)
    plain = X.AdamW([q], lr=0.1)
    assert plain.step() is None and plain.grad_norm is None


def test_norms_hold_their_own_words_only():
    # a kept or saved norm must not keep or save the scratch of its call
    p, g, m, v, _ = state_for([700_000, 5], torch.float32, 5)
    step = X.adamw_step_counter("cuda")
    total, each = X.gradient_norm(g, per_tensor=True)
    norms = [X.gradient_norm(g), total, X.clip_gradients_(g, 1e-3),
             X.adamw_update_(p, g, m, v, step, lr=0.1, max_norm=1.0),
             X.adamw_update_(p, g, m, v, step, lr=0.1, skip_nonfinite=True)]
    assert all(n.shape == () and n.untyped_storage().nbytes() == 4 for n in norms)
    assert each.untyped_storage().nbytes() == 8


def test_operators_stand_outside_autograd():
    # gradients with a graph of their own (create_graph): values are taken, no graph is built, and the documents say so
    x = torch.randn(3000, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(x.pow(3).sum(), x, create_graph=True)
    assert g.requires_grad
    total, each = X.gradient_norm([g], per_tensor=True)
    assert not total.requires_grad and not each.requires_grad
    h = g * 1.0
    assert not X.clip_gradients_([h], 1.0).requires_grad
    p, m, v = x.detach().clone().requires_grad_(), torch.zeros(3000, device="cuda"), torch.zeros(3000, device="cuda")
    assert not X.adamw_update_([p], [g], [m], [v], X.adamw_step_counter("cuda"), lr=0.1, max_norm=1.0).requires_grad
    for f in (X.gradient_norm, X.clip_gradients_, X.adamw_update_):
        assert "outside autograd" in " ".join(f.__doc__.split())


@pytest.mark.parametrize("eps", [1e-45, 1e-46, 1e-60, 1e-300])
def test_adamw_eps_below_32_bits(eps):
    # 0 / (0 + eps) is 0 for every eps above 0: an entry without gradient keeps its parameter
    p, m, v = make([3000], torch.float32, 1), make([3000], torch.float32, 2), make([3000], torch.float32, 3)
    g = [torch.zeros(3000, device="cuda")]
    m[0].zero_()
    v[0].zero_()
    before = p[0].clone()
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda"), lr=0.1, eps=eps)
    assert torch.equal(p[0], before)


@pytest.mark.parametrize("p", [2.0, 1.0])
@pytest.mark.parametrize("offset", [0, 1, 7, 31])
def test_same_bits_at_the_same_place_in_a_line(offset, p):
    # sums depend on lengths and on addresses modulo 128 bytes: what ranks have to agree on to agree in the last bit
    sizes = [1_000_003, 70_001, 400_000]
    data = make([sum(sizes)], torch.float32, 3)[0]
    norms = set()
    for lines in (0, 1, 5):
        flat = torch.empty(sum(sizes) + 32 * lines + offset, device="cuda")[32 * lines + offset:]
        flat.copy_(data)
        norms.add(float(X.gradient_norm(list(flat.split(sizes)), p)))
    assert len(norms) == 1


# ------------------------------- forms of the masked and mixed-type update --
KINDS = {  # parameter, gradient, master
    "f32": (torch.float32, torch.float32, False), "bf16": (torch.bfloat16, torch.bfloat16, False),
    "f16": (torch.float16, torch.float16, False), "bf16_master": (torch.bfloat16, torch.bfloat16, True),
    "f16_master": (torch.float16, torch.float16, True), "f32_f16grad": (torch.float32, torch.float16, False),
    "bf16_f32grad_master": (torch.bfloat16, torch.float32, True), "f16_bf16grad": (torch.float16, torch.bfloat16, False),
}


@pytest.mark.parametrize("name", ["some_empty", "vector_edges", "tile_edges", "leaves", "many"])
@pytest.mark.parametrize("kind", ["f16_master", "f32_f16grad", "bf16_f32grad_master", "f16_bf16grad"])
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_more_types(name, kind, clip):
    dtype, gdtype, mastered = KINDS[kind]
    p, g, m, v, masters = state_for(SIZE_SETS[name], dtype, 19, gdtype, mastered)
    old = [tuple(x.clone() for x in q) for q in zip(masters or p, g, m, v)]
    norm = norm64(g, 2)
    got = X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 4), lr=2e-3, weight_decay=0.02,
                          max_norm=0.2 * norm if clip else None, masters=masters)
    check_update(p, g, m, v, masters, old, 5, [2e-3] * len(p), (0.9, 0.999), 1e-8, 0.02,
                 0.2 * norm / (norm + CLIP_EPS) if clip else 1.0)
    assert got is None or abs(float(got) - norm) <= 10 * U * norm


@pytest.mark.parametrize("shape", [(3, 1), (5, 2), (1001, 2), (301, 3), (203, 5), (5, 16383), (5, 16384), (3, 20011),
                                   (2, 140_001), (40_000, 2), (30_011, 3), (60_001, 1), (7001, 48)])
@pytest.mark.parametrize("offsets", [(0, 0, 0, 0), (1, 1, 1, 1), (7, 7, 7, 7), (37, 37, 37, 37), (0, 1, 2, 3)])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_rows_at_offsets(shape, offsets, kind, clip):
    dtype, gdtype, mastered = KINDS[kind]
    n = math.prod(shape)
    p, g, m, v, masters = state_for([n + 64], dtype, 43, gdtype, mastered)
    whole = [p[0], g[0], m[0], v[0]] + ([masters[0]] if mastered else [])
    kept = [x.clone() for x in whole]
    places = list(offsets) + ([offsets[0]] if mastered else [])
    views = [[x[o:o + n].view(shape)] for x, o in zip(whole, places)]
    p, g, m, v = views[:4]
    masters = views[4] if mastered else None
    mask = torch.rand(shape[0], generator=torch.Generator().manual_seed(7)).lt(0.5).cuda()
    old = [tuple(x[0].clone() for x in (masters or p, g, m, v))]
    bits = p[0].clone()
    norm = norm64(g, 2)
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 9), lr=0.01, row_mask=mask, masters=masters,
                    max_norm=0.5 * norm if clip else None)
    check_update(p, g, m, v, masters, old, 10, [0.01], (0.9, 0.999), 1e-8, 0.0,
                 0.5 * norm / (norm + CLIP_EPS) if clip else 1.0, [mask])
    assert torch.equal(p[0][~mask], bits[~mask])
    for x, k, o in zip(whole, kept, places):  # the bytes around each view
        assert torch.equal(x[:o], k[:o]) and torch.equal(x[o + n:], k[o + n:])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16_master"])
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_rows_large_at_offsets(kind, clip):
    # more tiles than blocks, tensors masked and not, at offsets of their own in one buffer for each array
    dtype, gdtype, mastered = KINDS[kind]
    shapes = [(1_000_003, 3), (1_000_003,), (400_001, 2), (129, 20_011), (300_007,)]
    sizes = [math.prod(s) for s in shapes]
    flat = state_for([sum(sizes) + 5], dtype, 47, gdtype, mastered)

    def split(x):
        return [y.view(s) for y, s in zip(x[0][5:].split(sizes), shapes)]

    p, g, m, v = (split(x) for x in flat[:4])
    masters = split(flat[4]) if mastered else None
    masks = [torch.rand(s[0], generator=torch.Generator().manual_seed(i)).lt(0.4).cuda() if i != 4 else None
             for i, s in enumerate(shapes)]
    old = [tuple(x.clone() for x in q) for q in zip(masters or p, g, m, v)]
    bits = [x.clone() for x in p]
    norm = norm64(g, 2)
    X.adamw_update_(p, g, m, v, X.adamw_step_counter("cuda", 9), lr=0.01, row_mask=masks, masters=masters,
                    max_norm=0.5 * norm if clip else None)
    check_update(p, g, m, v, masters, old, 10, [0.01] * 5, (0.9, 0.999), 1e-8, 0.0,
                 0.5 * norm / (norm + CLIP_EPS) if clip else 1.0, masks)
    for x, b, mask in zip(p, bits, masks):
        assert mask is None or torch.equal(x[~mask], b[~mask])
