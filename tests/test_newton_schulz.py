"""Newton-Schulz on caller-owned matrices (vb_orthogonalize, vb_muon_multi_tensor_step) against the
formulas in 64 bits:

    X_0 = U / (|U|_F + eps);  X_{k+1} = a X_k + b (X_k X_k^T) X_k + c (X_k X_k^T)^2 X_k;  O = X_K
    v <- mu v + g;  u = g + mu v or v;  p <- p (1 - lr wd) - lr s O(u)

Tolerance of O.  Rounding a stored matrix M to a relative u per element moves it by at most u |M|_F.  Such a
move of the iterate X_k reaches O through the remaining steps, each of which stretches by at most L_j, the
largest |d/dx x q_j(x^2)| on the singular values' range.  A step stores at most six matrices (X, G, R, T, P,
the next G); a relative move of one of the short-side ones moves the iterate by no more than a few times
that, since q and its terms are bounded by 3 max|q|.  So

    |dO|_F <= sum_k 6 * 3 * u |X_k|_F prod_{j >= k} L_j

computed below from the exact iterates.  u is 2^-11 for f16 (half a step, 2^-11 relative to the value) and for two
planes 2^-22, to which the tensor core's truncating f32 accumulation adds 2^-23 per 16-wide product that enters a
sum.  The result's own rounding is added per element: eps / 2 of its type.
"""
import ctypes as C
import math

import numpy as np
import pytest

QUINTIC = [(3.4445, -4.7750, 2.0315)] * 5
CUBIC = [(1.5, -0.5, 0.0)] * 5
MIXED = [(8.0, -22.0, 16.0), (4.0, -2.9, 0.55), (1.5, -0.5, 0.0), (3.3, -2.4, 0.48)]


# ---- host only ---------------------------------------------------------------------------------

def _products(rows, cols, coefficients, mode=3):
    from volta_b200 import plan_newton_schulz
    return plan_newton_schulz(rows, cols, coefficients, mode)


def _run_schedule(products, x0, coefficients):
    """The planned products in float64, powers of two and all."""
    n = x0.shape[0]
    scale = 1.0 / np.linalg.norm(x0)
    buffers = {0: x0.copy()}
    stages = sorted({p["stage"] for p in products})
    for s in stages:
        written = {}
        for p in (p for p in products if p["stage"] == s):
            a, b = buffers[p["A"]], buffers[p["B"]]
            acc = a @ b if p["update"] else a @ b.T
            assert acc.shape == (n, b.shape[1] if p["update"] else n)
            d = p["g"] * acc
            if p["E"] >= 0:
                d = d + p["e"] * buffers[p["E"]]
            if p["F"] >= 0:
                d = d + p["f"] * buffers[p["F"]]
            assert p["D"] not in written and p["D"] not in (p["A"], p["B"], p["E"], p["F"])
            written[p["D"]] = d * scale ** p["scale_power"]
        read = {p[k] for p in products if p["stage"] == s for k in "ABEF"}
        assert not read & set(written), "a stage overwrites what it reads"
        buffers.update(written)
        for d in written.values():
            assert np.abs(d).max() < 32768  # inside f16 with room for noise
    return buffers


@pytest.mark.parametrize("mode", [3, 2], ids=["f16", "f32"])
@pytest.mark.parametrize("shape", [(24, 24), (16, 80), (80, 16), (1, 7), (1, 1), (33, 48), (70, 70), (300, 72)])
@pytest.mark.parametrize("coefficients", [QUINTIC, CUBIC, MIXED, QUINTIC[:1], CUBIC[:2], [(1.0, 0.0, 0.0)],
                                          [(2.0, -1.5, 0.5)] * 12])
def test_planned_products_are_the_iteration(shape, coefficients, mode):
    rng = np.random.default_rng(3)
    u = rng.standard_normal(shape)
    x = u.T if shape[0] > shape[1] else u
    products, final_scale = _products(*shape, coefficients, mode)
    out = _run_schedule(products, x, coefficients)
    want = x / np.linalg.norm(x)
    for a, b, c in coefficients:
        g = want @ want.T
        want = a * want + (b * g + c * g @ g) @ want
    got = out[products[-1]["D"]] * final_scale
    # f64 products; the coefficients pass through f32
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


def test_groups_follow_the_amplification_limits():
    """Long matrices: the quintic runs in groups of 3 and 2 (of 2, 2 and 1 where the short side is small), square
    ones step by step, the cubic as one; short sides of at most 64 as one group in f16, in pairs to f32 accuracy."""
    grams = lambda shape, co, mode=3: [p["stage"] for p in _products(*shape, co, mode)[0] if p["gram"]]  # noqa: E731
    assert len(grams((1024, 256), QUINTIC)) == 2
    assert len(grams((100, 256), QUINTIC)) == 3
    assert len(grams((100, 100), QUINTIC)) == 5
    assert len(grams((256, 100), CUBIC)) == 1
    assert len(grams((64, 256), QUINTIC)) == 1
    assert len(grams((64, 256), QUINTIC, 2)) == 3


def test_plan_refuses_without_a_device_call():
    from volta_b200 import VoltaB200Error, _lib
    h = C.c_void_p()
    ok = (C.c_float * 3)(1.5, -0.5, 0.0)
    one = (C.c_int64 * 1)(4)
    with pytest.raises(VoltaB200Error, match="engine is null"):
        _lib.call("vb_ns_plan_create", None, 1, one, one, 1, ok, 1e-7, 3, C.byref(h))
    with pytest.raises(VoltaB200Error, match="plan is null"):
        _lib.call("vb_orthogonalize", None, None, None)
    with pytest.raises(VoltaB200Error, match="plan is null"):
        _lib.call("vb_muon_multi_tensor_step", None, None, None, None, None, None)
    with pytest.raises(VoltaB200Error, match="plan is null"):
        _lib.call("vb_ns_matrices_create", None, 0, None, None, C.byref(h))
    for bad in ([(float("nan"), 0, 0)], [(1e9, 0.0, 0.0)], [(3.0, 5.0, 5.0)] * 8):
        with pytest.raises(VoltaB200Error):
            _products(8, 8, bad)


def test_strides_of_a_matrix_view():
    from volta_b200.newton_schulz import _two_strides
    assert _two_strides((5, 7), (7, 1)) == (7, 1)
    assert _two_strides((5, 7), (1, 5)) == (1, 5)
    assert _two_strides((8, 3, 3, 3), (27, 9, 3, 1)) == (27, 1)
    assert _two_strides((8, 1, 3, 3), (9, 777, 3, 1)) == (9, 1)
    assert _two_strides((8, 4, 1), (4, 1, 5)) == (4, 1)
    assert _two_strides((6,), (2,)) == (2, 1)
    with pytest.raises(ValueError):
        _two_strides((8, 3, 4), (24, 8, 1))


# ---- on the device -----------------------------------------------------------------------------

gpu = pytest.mark.gpu


def _exact(u, coefficients, eps=1e-7):
    """(O, bound on |dO|_F per unit of u) of one float64 matrix on the device."""
    import torch
    x = u.mT if u.shape[0] > u.shape[1] else u
    x = x / (torch.linalg.norm(x) + eps)
    norms, stretch = [], []
    top = 1.0
    for a, b, c in coefficients:
        norms.append(torch.linalg.norm(x).item())
        t = np.linspace(0.0, top, 2001)
        stretch.append(np.abs(a + 3 * b * t ** 2 + 5 * c * t ** 4).max())
        top = np.abs(a * t + b * t ** 3 + c * t ** 5).max()
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    bound = sum(18.0 * norms[k] * math.prod(stretch[k:]) for k in range(len(norms)))
    return (x.mT if u.shape[0] > u.shape[1] else x), bound


def _unit(mode, shape):
    from volta_b200 import VB_NS_F16
    n, m = min(shape), max(shape)
    return 2.0 ** -11 if mode == VB_NS_F16 else 2.0 ** -22 + 2.0 ** -23 * 3 * (m + n) / 16


def _gradient(torch, shape, seed, dtype, noise=0.3, scale=1e-3):
    gen = torch.Generator(device="cuda:0").manual_seed(seed)
    rank = max(1, min(shape) // 16)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda:0")  # noqa: E731
    return (scale * (r(shape[0], rank) @ r(rank, shape[1]) / rank ** 0.5 + noise * r(*shape))).to(dtype)


def _strided(torch, x, layout):
    """The same matrix in other memory: rows, transposed, a block of a wider matrix, every third element, unaligned."""
    r, c = x.shape
    if layout == "rows":
        return x.clone()
    if layout == "transposed":
        return x.t().contiguous().t()
    if layout == "block":
        wide = torch.zeros(r, c + 24, dtype=x.dtype, device=x.device)
        view = wide[:, 8:8 + c]
    elif layout == "sparse":
        view = torch.zeros(r, 2, c, 3, dtype=x.dtype, device=x.device)[:, 1, :, 1]
    elif layout == "offset":
        view = torch.zeros(r * c + 1, dtype=x.dtype, device=x.device)[1:].view(r, c)
    view.copy_(x)
    return view


def _close(got, want, bound, unit, dtype):
    """|got - want|_F against the bound, plus the rounding of the result to its type."""
    import torch
    off = torch.linalg.norm(got.double() - want).item()
    half = 0.0 if dtype is None else torch.finfo(dtype).eps / 2
    limit = bound * unit + half * torch.linalg.norm(want).item() + 1e-30
    assert math.isfinite(off) and off <= limit, (off, limit, torch.linalg.norm(want).item())


SHAPES = [(1, 1), (1, 5), (7, 1), (2, 2), (9, 32), (64, 288), (10, 128), (127, 129), (128, 128), (129, 127), (256, 784),
          (200, 1000), (513, 1000), (1024, 64), (300, 300), (640, 384)]


@gpu
@pytest.mark.parametrize("mode", ["f16", "f32"])
@pytest.mark.parametrize("coefficients", [QUINTIC, MIXED, CUBIC], ids=["quintic", "mixed", "cubic"])
def test_orthogonalize_ragged_list(engine, mode, coefficients):
    import torch
    import volta_b200 as vb
    ns_mode, dtype = (vb.VB_NS_F16, torch.bfloat16) if mode == "f16" else (vb.VB_NS_F32_TC, torch.float32)
    plan = vb.NewtonSchulzPlan(SHAPES, coefficients, ns_mode=ns_mode, engine=engine)
    xs = [_gradient(torch, s, 10 + i, dtype) for i, s in enumerate(SHAPES)]
    outs = [torch.full(s, 7.0, dtype=dtype, device="cuda:0") for s in SHAPES]
    torch.cuda.synchronize()
    plan.orthogonalize(xs, outs)
    engine.synchronize()
    for x, o, s in zip(xs, outs, SHAPES):
        want, bound = _exact(x.double(), coefficients)
        _close(o, want, bound, _unit(ns_mode, s), dtype)


@gpu
@pytest.mark.parametrize("shape", [(2048, 1024), (1024, 1536), (1000, 4097), (2049, 2047)])
@pytest.mark.parametrize("mode", ["f16", "f32"])
def test_orthogonalize_large(engine, shape, mode):
    import torch
    import volta_b200 as vb
    ns_mode, dtype = (vb.VB_NS_F16, torch.float16) if mode == "f16" else (vb.VB_NS_F32_TC, torch.float32)
    plan = vb.NewtonSchulzPlan([shape] * 2, QUINTIC, ns_mode=ns_mode, engine=engine)
    xs = [_gradient(torch, shape, 50 + i, dtype, scale=1.0) for i in range(2)]
    outs = [torch.empty_like(x) for x in xs]
    torch.cuda.synchronize()
    plan.orthogonalize(xs, outs)
    engine.synchronize()
    for x, o in zip(xs, outs):
        want, bound = _exact(x.double(), QUINTIC)
        _close(o, want, bound, _unit(ns_mode, shape), dtype)


@gpu
@pytest.mark.parametrize("kinds", [("float32", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("layouts", [("rows", "transposed"), ("transposed", "block"), ("block", "sparse"),
                                     ("sparse", "offset"), ("offset", "rows"), ("transposed", "transposed")])
@pytest.mark.parametrize("shape", [(45, 130), (130, 45), (64, 256)])
def test_orthogonalize_types_and_strides(engine, shape, layouts, kinds):
    import torch
    import volta_b200 as vb
    ti, to = (getattr(torch, k) for k in kinds)
    plan = vb.NewtonSchulzPlan([shape], QUINTIC, engine=engine)
    x = _strided(torch, _gradient(torch, shape, 5, ti), layouts[0])
    o = _strided(torch, torch.full(shape, 9.0, dtype=to, device="cuda:0"), layouts[1])
    around = o._base.clone() if o._base is not None else None
    torch.cuda.synchronize()
    plan.orthogonalize([x], [o])
    engine.synchronize()
    want, bound = _exact(x.double(), QUINTIC)
    _close(o, want, bound, _unit(vb.VB_NS_F16, shape), to)
    if around is not None:  # elements between the matrix's own are left as they were
        o.fill_(9.0)
        assert torch.equal(o._base, around)


@gpu
@pytest.mark.parametrize("mode", ["f16", "f32"])
@pytest.mark.parametrize("shape", [(96, 160), (48, 100), (200, 30), (300, 70)])
def test_orthogonalize_in_place_zero_tiny_huge_and_undefined(engine, shape, mode):
    import torch
    import volta_b200 as vb
    ns_mode = vb.VB_NS_F32_TC if mode == "f32" else vb.VB_NS_F16
    base = _gradient(torch, shape, 1, torch.float32)
    xs = [torch.zeros(shape, device="cuda:0"), base * 1e-30, base * 1e30, base.clone(), base.clone(), base * 1e-9]
    xs[3][5, 7] = float("inf")
    xs[4][0, 0] = float("nan")
    plan = vb.NewtonSchulzPlan([shape] * 6, QUINTIC, eps=1e-12, ns_mode=ns_mode, engine=engine)
    before = [x.clone() for x in xs]
    torch.cuda.synchronize()
    table = plan.matrices(xs)
    plan.orthogonalize(table, table)
    engine.synchronize()
    assert torch.equal(xs[0], before[0])
    # U far below eps: O = prod(a) U / eps, in f16 with an absolute floor of 2^-25 2^-12 per element
    want, _ = _exact(before[1].double(), QUINTIC, 1e-12)
    assert (xs[1].double() - want).abs().max().item() <= 2.0 ** -36
    for k, eps in ((2, 1e-12), (5, 1e-12)):
        want, bound = _exact(before[k].double(), QUINTIC, eps)
        _close(xs[k], want, bound, _unit(ns_mode, shape), torch.float32)
    assert torch.isnan(xs[3]).all() and torch.isnan(xs[4]).all()


@gpu
@pytest.mark.parametrize("mode", ["f16", "f32"])
@pytest.mark.parametrize("coefficients", [QUINTIC[:1], [(2.0, -1.5, 0.5)] * 12, [(1.0, 0.0, 0.0)] * 2, [(1.5, -0.5, 0.0)] * 20,
                                          [(1.0, 0.0, 1e-20)] * 40, [(1.9, 0.0, 0.0)] * 6],
                         ids=["one", "twelve", "identity", "twenty linear", "more than a small program holds", "growing"])
def test_other_step_counts(engine, coefficients, mode):
    import torch
    import volta_b200 as vb
    shapes = [(40, 90), (150, 150), (129, 700)]
    ns_mode = vb.VB_NS_F32_TC if mode == "f32" else vb.VB_NS_F16
    plan = vb.NewtonSchulzPlan(shapes, coefficients, ns_mode=ns_mode, engine=engine)
    xs = [_gradient(torch, s, 20 + i, torch.float32) for i, s in enumerate(shapes)]
    outs = [torch.empty_like(x) for x in xs]
    torch.cuda.synchronize()
    plan.orthogonalize(xs, outs)
    engine.synchronize()
    for x, o, s in zip(xs, outs, shapes):
        want, bound = _exact(x.double(), coefficients)
        _close(o, want, bound, _unit(ns_mode, s), torch.float32)


@gpu
@pytest.mark.parametrize("mode", ["f16", "f32"])
@pytest.mark.parametrize("shapes", [[(100, 4100)], [(4500, 128), (65, 2100)], [(20, 30)] * 210, [(70, 90)] * 130 + [(30, 9)] * 3,
                                    [(512, 512)] * 40 + [(100, 700), (600, 1300), (1, 3)], [(64, 9000), (9000, 3)]],
                         ids=["long", "tall", "many small", "many", "pairs", "very long"])
def test_lists_of_every_kind(engine, shapes, mode):
    """Contractions cut into pieces, several launches of small matrices, tile pairs with half-empty edges, columns
    that do not fit one cluster."""
    import torch
    import volta_b200 as vb
    ns_mode, dtype = (vb.VB_NS_F32_TC, torch.float32) if mode == "f32" else (vb.VB_NS_F16, torch.bfloat16)
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, ns_mode=ns_mode, engine=engine)
    xs = [_gradient(torch, s, 70 + i, dtype) for i, s in enumerate(shapes)]
    outs = [torch.empty_like(x) for x in xs]
    torch.cuda.synchronize()
    plan.orthogonalize(xs, outs)
    engine.synchronize()
    for x, o, s in zip(xs, outs, shapes):
        want, bound = _exact(x.double(), QUINTIC)
        _close(o, want, bound, _unit(ns_mode, s), dtype)


@gpu
def test_offsets_beyond_32_bits(engine):
    """Rows 1.1e9 elements apart: element offsets pass 2^31 in inputs, outputs, velocities and parameters."""
    import torch
    import volta_b200 as vb
    pitch = 1_100_000_000
    big = torch.zeros(3 * pitch, dtype=torch.bfloat16, device="cuda:0")
    for shape, at in (((3, 40), 0), ((3, 40), pitch // 2)):
        x = big.as_strided(shape, (pitch, 1), at)
        x.copy_(_gradient(torch, shape, 4, torch.bfloat16))
    wide = big.as_strided((3, 40), (pitch, 1), 0)
    tall = big.as_strided((40, 3), (1, pitch), pitch // 2)
    for x in (wide, tall):
        plan = vb.NewtonSchulzPlan([x.shape], QUINTIC, engine=engine)
        before = x.clone()
        torch.cuda.synchronize()
        plan.orthogonalize([x], [x])
        engine.synchronize()
        want, bound = _exact(before.double(), QUINTIC)
        _close(x, want, bound, _unit(vb.VB_NS_F16, x.shape), torch.bfloat16)
    # and through the general path: two rows of 130 columns, 130 rows of 70
    plan = vb.NewtonSchulzPlan([(70, 130)], QUINTIC, engine=engine)
    view = big.as_strided((70, 130), (40_000_000, 1), 0)
    view.copy_(_gradient(torch, (70, 130), 6, torch.bfloat16))
    before, velocity = view.clone(), torch.zeros(70, 130, device="cuda:0")
    grad = _gradient(torch, (70, 130), 7, torch.bfloat16)
    torch.cuda.synchronize()
    plan.muon_step([view], [grad], [velocity], lr=0.1, momentum=0.0, nesterov=False)
    engine.synchronize()
    o, bound = _exact(grad.double(), QUINTIC)
    want = before.double() - float(np.float32(0.1)) * o
    off = torch.linalg.norm(view.double() - want).item()
    assert off <= 0.1 * bound * _unit(vb.VB_NS_F16, (70, 130)) + 2.0 ** -8 * torch.linalg.norm(want).item()


@gpu
def test_same_bits_every_call_and_in_other_company(engine):
    """Nothing is kept from one call for the next, and a matrix's result does not hang on the list it is in."""
    import torch
    import volta_b200 as vb
    shapes = [(256, 512), (100, 40), (256, 512)]
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, engine=engine)
    runs = []
    for seed in (1, 2, 1):
        xs = [_gradient(torch, s, seed + i, torch.bfloat16) for i, s in enumerate(shapes)]
        outs = [torch.empty_like(x) for x in xs]
        torch.cuda.synchronize()
        plan.orthogonalize(xs, outs)
        runs.append(outs)
    engine.synchronize()
    for a, b, c in zip(*runs):
        assert torch.equal(a, c) and not torch.equal(a, b)


def _step_case(torch, shapes, kinds, layouts, seed=0):
    tp, tg, tv = (getattr(torch, k) for k in kinds)
    p = [_strided(torch, (torch.randn(s, generator=torch.Generator("cuda:0").manual_seed(seed + i), device="cuda:0") * 0.05).to(tp), layouts[0])
         for i, s in enumerate(shapes)]
    g = [_strided(torch, _gradient(torch, s, seed + 100 + i, tg), layouts[1]) for i, s in enumerate(shapes)]
    v = [_strided(torch, _gradient(torch, s, seed + 200 + i, tv, scale=4e-3), layouts[2]) for i, s in enumerate(shapes)]
    return p, g, v


@gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("kinds", [("float32", "float32", "float32"), ("float32", "bfloat16", "float32"),
                                   ("bfloat16", "bfloat16", "bfloat16"), ("bfloat16", "float16", "float32")])
@pytest.mark.parametrize("layouts", [("rows", "rows", "rows"), ("rows", "transposed", "rows"),
                                     ("transposed", "rows", "block"), ("offset", "sparse", "transposed")])
def test_muon_step(engine, kinds, layouts, nesterov):
    import torch
    import volta_b200 as vb
    shapes = [(130, 70), (70, 130), (1, 9), (256, 257), (64, 300)]
    mode = vb.VB_NS_F32_TC if kinds[1] == "float32" else vb.VB_NS_F16
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, ns_mode=mode, engine=engine)
    p, g, v = _step_case(torch, shapes, kinds, layouts)
    p0, v0 = [x.double() for x in p], [x.double() for x in v]
    scales = [0.5 + 0.25 * i for i in range(len(shapes))]
    lr, mu, wd = 0.02, 0.9, 0.1
    torch.cuda.synchronize()
    plan.muon_step(p, g, v, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scales=scales)
    engine.synchronize()
    for i, s in enumerate(shapes):
        mu32, lr32, wd32 = (float(np.float32(z)) for z in (mu, lr, wd))
        want_v = mu32 * v0[i] + g[i].double()
        tv = getattr(torch, kinds[2])
        # one fma in f32 and the rounding to the array's type, element by element
        limit = (torch.finfo(tv).eps / 2 + 2.0 ** -23) * want_v.abs() + 1e-30
        assert ((v[i].double() - want_v).abs() <= limit).all()
        u = g[i].double() + mu32 * want_v if nesterov else want_v
        o, bound = _exact(u, QUINTIC)
        # u in f32 (two fmas, 2^-24 each of terms no larger than 2 |u| here) joins the first iterate's rounding
        unit = _unit(mode, s) + 2.0 ** -22
        want_p = p0[i] * (1.0 - lr32 * wd32) - lr32 * scales[i] * o
        tp = getattr(torch, kinds[0])
        off = torch.linalg.norm(p[i].double() - want_p).item()
        limit = lr * scales[i] * bound * unit + (torch.finfo(tp).eps / 2 + 2.0 ** -22) * torch.linalg.norm(want_p).item()
        assert off <= limit, (i, off, limit)


@gpu
def test_muon_step_skips_absent_gradients(engine):
    import torch
    import volta_b200 as vb
    shapes = [(64, 96), (200, 150), (33, 17)]
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, engine=engine)
    p, g, v = _step_case(torch, shapes, ("float32",) * 3, ("rows",) * 3)
    p1, v1 = [x.clone() for x in p], [x.clone() for x in v]
    torch.cuda.synchronize()
    plan.muon_step(p, [g[0], None, g[2]], v, lr=0.1)
    engine.synchronize()
    alone = vb.NewtonSchulzPlan([shapes[0], shapes[2]], QUINTIC, engine=engine)
    assert torch.equal(p[1], p1[1]) and torch.equal(v[1], v1[1])
    alone.muon_step([p1[0], p1[2]], [g[0], g[2]], [v1[0], v1[2]], lr=0.1)
    engine.synchronize()
    for k in (0, 2):
        assert torch.equal(p[k], p1[k]) and torch.equal(v[k], v1[k])
    before = [x.clone() for x in p + v]
    plan.muon_step(p, [None] * 3, v, lr=0.1)  # no gradient at all
    engine.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, p + v))
    plan.muon_step(p, g, v, lr=0.1)           # and all of them again
    engine.synchronize()
    assert not any(torch.equal(a, b) for a, b in zip(before, p + v))


@gpu
def test_muon_step_is_the_reference_step(engine, oracle):
    """With the cubic, scale 0.1 and no weight decay the step is Volta's Muon::step."""
    import torch
    import volta_b200 as vb
    shapes = [(48, 96), (130, 64), (36, 36)]
    rng = np.random.default_rng(5)
    p = [(rng.standard_normal(s) * 0.05).astype(np.float32) for s in shapes]
    ref = oracle.Muon([x.copy() for x in p], 0.1, 0.9, True, 5)
    dev = [torch.from_numpy(x.copy()).cuda() for x in p]
    vel = [torch.zeros_like(x) for x in dev]
    plan = vb.NewtonSchulzPlan(shapes, CUBIC, eps=0.0, ns_mode=vb.VB_NS_F32_TC, engine=engine)
    for s in range(3):
        g = [(rng.standard_normal(x) * 1e-1).astype(np.float32) for x in shapes]
        ref.step(g)
        gd = [torch.from_numpy(x).cuda() for x in g]
        torch.cuda.synchronize()
        plan.muon_step(dev, gd, vel, lr=0.1, momentum=0.9, scales=[0.1] * 3)
        engine.synchronize()
    for got, want, start in zip(dev, ref.params, p):
        # the update's share of the weights: 3 steps of lr 0.1 * 0.1 * |O| with O to 1e-5, eps of the norm 1e-8 / |u|^2
        off = np.linalg.norm(got.cpu().numpy().astype(np.float64) - want)
        assert off <= 3 * 0.01 * 1e-5 * math.sqrt(min(want.shape)) + 4 * 2.0 ** -24 * np.linalg.norm(want)


@gpu
def test_orthogonalize_then_step_together(engine):
    """A run of both operators on one plan, as a program has them: the step equals the pieces."""
    import torch
    import volta_b200 as vb
    shapes = [(256, 128), (100, 300)]
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, ns_mode=vb.VB_NS_F32_TC, engine=engine)
    p, g, v = _step_case(torch, shapes, ("float32",) * 3, ("rows",) * 3, seed=9)
    pp, vv = [x.clone() for x in p], [x.clone() for x in v]
    o = [torch.empty_like(x) for x in p]
    stream = torch.cuda.ExternalStream(engine.stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(3):
            u = []
            for k in range(2):
                vv[k].mul_(0.9).add_(g[k])
                u.append(g[k] + 0.9 * vv[k])
            plan.orthogonalize(u, o)
            for k in range(2):
                pp[k].mul_(1 - 0.01 * 0.1).sub_(0.01 * o[k])
            plan.muon_step(p, g, v, lr=0.01, momentum=0.9, weight_decay=0.1)
    engine.synchronize()
    for k in range(2):
        # v: fma against product and sum, half a step of f32 each time
        assert (v[k] - vv[k]).abs().max().item() <= 3 * 2.0 ** -23 * v[k].abs().max().item()
        _, bound = _exact(u[k].double(), QUINTIC)
        off = torch.linalg.norm(p[k].double() - pp[k].double()).item()
        assert off <= 3 * (0.01 * bound * _unit(vb.VB_NS_F32_TC, shapes[k]) + 2.0 ** -22 * torch.linalg.norm(pp[k]).item())


@gpu
def test_captured_calls_replay(engine):
    """Both operators captured from the engine's stream; replayed on new contents of the same buffers."""
    import torch
    import volta_b200 as vb
    shapes = [(128, 200), (64, 64), (300, 140)]
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, engine=engine)
    p, g, v = _step_case(torch, shapes, ("float32",) * 3, ("rows",) * 3)
    o = [torch.empty_like(x) for x in p]
    tp, tg, tv, to = (plan.matrices(x) for x in (p, g, v, o))
    fresh = [x.clone() for x in p + v]
    stream = torch.cuda.ExternalStream(engine.stream)
    plan.orthogonalize(tg, to)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan.orthogonalize(tg, to)
        plan.muon_step(tp, tg, tv, lr=0.05)
    for seed in (300, 400):
        for x, y in zip(p + v, fresh):
            x.copy_(y)
        for i, x in enumerate(g):
            x.copy_(_gradient(torch, x.shape, seed + i, torch.float32))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in o + p + v]
        for x, y in zip(p + v, fresh):
            x.copy_(y)
        torch.cuda.synchronize()
        plan.orthogonalize(tg, to)
        plan.muon_step(tp, tg, tv, lr=0.05)
        engine.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, o + p + v))


@gpu
@pytest.mark.parametrize("others", [[], [(200, 300)]], ids=["small only", "beside a larger one"])
def test_launches_side_by_side_are_ordered_with_the_engine(engine, others):
    """300 small matrices are several launches that run beside each other: the call sees what the stream wrote before
    it and is complete for what the stream does next, at once and as a replayed graph."""
    import torch
    import volta_b200 as vb
    shapes = [(96, 40)] * 300 + others
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, engine=engine)
    x, mid, out = ([torch.zeros(s, device="cuda") for s in shapes] for _ in range(3))
    tx, tm, to = (plan.matrices(a) for a in (x, mid, out))
    want = []
    stream = torch.cuda.ExternalStream(engine.stream)
    source = [[_gradient(torch, s, 1000 * k + i, torch.float32) for i, s in enumerate(shapes)] for k in range(3)]
    for fresh in source:  # one call at a time
        torch._foreach_copy_(x, fresh)
        torch.cuda.synchronize()
        plan.orthogonalize(tx, tm)
        engine.synchronize()
        plan.orthogonalize(tm, to)
        engine.synchronize()
        want.append([o.clone() for o in out])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        plan.orthogonalize(tx, tm)
        plan.orthogonalize(tm, to)
    got = []
    with torch.cuda.stream(stream):
        for k, fresh in enumerate(source + source):  # nothing waits on the host in between
            torch._foreach_copy_(x, fresh)
            if k < len(source):
                plan.orthogonalize(tx, tm)
                plan.orthogonalize(tm, to)
            else:
                graph.replay()
            got.append([o.clone() for o in out])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want + want) for a, b in zip(g, w))
    plan.close()


@gpu
def test_refusals(engine):
    import torch
    import volta_b200 as vb
    from volta_b200 import VoltaB200Error
    E = VoltaB200Error
    plan = vb.NewtonSchulzPlan([(8, 16), (4, 4)], QUINTIC, engine=engine)
    make = lambda *s: torch.zeros(*s, device="cuda:0")  # noqa: E731
    a, b = make(8, 16), make(4, 4)
    for bad in (dict(ns_mode=vb.VB_NS_BF16), dict(ns_mode=vb.VB_NS_F32), dict(ns_mode=77), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(E):
            vb.NewtonSchulzPlan([(8, 16)], QUINTIC, engine=engine, **bad)
    with pytest.raises(E):
        vb.NewtonSchulzPlan([(8, 16)], [], engine=engine)
    with pytest.raises(E):
        vb.NewtonSchulzPlan([(8, 65537)], QUINTIC, engine=engine)
    with pytest.raises(ValueError):
        plan.matrices([a])
    with pytest.raises(ValueError):
        plan.matrices([a.t(), b])
    with pytest.raises(TypeError):
        plan.matrices([a.double(), b])
    with pytest.raises(TypeError):
        plan.matrices([a, b.half()])
    with pytest.raises((E, ValueError)):
        plan.matrices([a.cpu(), b])
    with pytest.raises(E, match="null"):
        plan.orthogonalize([a, None], [a, b])
    with pytest.raises(E, match="share"):
        plan.orthogonalize([a, b], [make(1, 16).expand(8, 16), b])
    c = make(8, 16)
    with pytest.raises(E, match="one address"):
        vb.NewtonSchulzPlan([(8, 16)] * 2, QUINTIC, engine=engine).orthogonalize([a, c], [c, c])
    square = make(4, 4)
    with pytest.raises(E, match="one address"):
        plan.orthogonalize([a, square], [c, square.t()])
    with pytest.raises(E, match="one address"):
        plan.muon_step([a, b], [a, make(4, 4)], [c, make(4, 4)], lr=0.1)
    with pytest.raises(E, match="finite"):
        plan.muon_step([a, b], [c, make(4, 4)], [make(8, 16), make(4, 4)], lr=float("nan"))
    with pytest.raises(ValueError):
        plan.muon_step([a, b], [c, make(4, 4)], [make(8, 16), make(4, 4)], lr=0.1, scales=[1.0])
    other = vb.NewtonSchulzPlan([(8, 16), (4, 4)], QUINTIC, engine=engine)
    with pytest.raises(E, match="another plan"):
        plan.orthogonalize(other.matrices([a, b]), plan.matrices([c, square]))
    # reading a broadcast input is fine, and so are empty plans and matrices without elements
    plan.orthogonalize([make(1, 16).expand(8, 16), b], [c, square])
    empty = vb.NewtonSchulzPlan([], QUINTIC, engine=engine)
    empty.orthogonalize([], [])
    hollow = vb.NewtonSchulzPlan([(0, 5), (3, 4)], QUINTIC, engine=engine)
    out = make(3, 4)
    hollow.orthogonalize([make(0, 5), make(3, 4) + 1], [make(0, 5), out])
    engine.synchronize()
    assert out.abs().max().item() > 0


@gpu
def test_arrays_of_another_matrix_are_refused(engine):
    """Matrices of one call run at the same time, so none may write what another reads."""
    import torch
    import volta_b200 as vb
    plan = vb.NewtonSchulzPlan([(8, 16), (8, 16)], QUINTIC, engine=engine)
    a, b, c, d, e, f = (torch.ones(8, 16, device="cuda:0") for _ in range(6))
    torch.cuda.synchronize()
    for x, o in (([a, b], [b, a]), ([a, a], [a, b]), ([a, b], [c, a]), ([a, b], [b.t().t(), c])):
        with pytest.raises(vb.VoltaB200Error, match="one address"):
            plan.orthogonalize(x, o)
    for p, g, v in (([a, b], [c, a], [d, e]), ([a, b], [c, d], [e, c]), ([a, b], [c, d], [b, e]), ([a, b], [None, a], [d, e])):
        with pytest.raises(vb.VoltaB200Error, match="one address"):
            plan.muon_step(p, g, v, lr=0.1)
    plan.orthogonalize([a, a], [c, d])  # one input read twice
    plan.orthogonalize([a, b], [a, c])  # in place
    plan.muon_step([a, b], [c, c], [e, f], lr=0.1)
    engine.synchronize()
    assert torch.equal(e, f)


@gpu
def test_a_list_does_not_outlive_its_plan(engine):
    """A plan that takes the place of a closed one does not accept the closed one's lists."""
    import torch
    import volta_b200 as vb
    x, y = torch.ones(8, 16, device="cuda:0"), torch.ones(8, 16, device="cuda:0")
    torch.cuda.synchronize()
    addresses, lists, back = set(), [], False
    for _ in range(100):
        plan = vb.NewtonSchulzPlan([(8, 16)], QUINTIC, engine=engine)
        back = back or plan._h.value in addresses
        addresses.add(plan._h.value)
        for old in lists:
            with pytest.raises(vb.VoltaB200Error, match="another plan"):
                plan.orthogonalize(old, [y])
        lists.append(plan.matrices([x]))
        plan.orthogonalize(lists[-1], [y])
        plan.close()
        if back:  # an allocator may also never give an address twice
            break


@gpu
@pytest.mark.parametrize("mode", ["f16", "f32"])
@pytest.mark.parametrize("columns", [1, 3, 8, 20])
@pytest.mark.parametrize("rows", [1, 5, 77, 300])
def test_leading_columns_of_a_wider_array(engine, rows, columns, mode):
    """x[:, :k] of a contiguous array whose rows are 16-byte aligned: what lies behind the k columns stays."""
    import torch
    import volta_b200 as vb
    ns_mode, dtype = (vb.VB_NS_F32_TC, torch.float32) if mode == "f32" else (vb.VB_NS_F16, torch.bfloat16)
    shape = (rows, columns)
    plan = vb.NewtonSchulzPlan([shape, shape, shape[::-1]], QUINTIC, ns_mode=ns_mode, engine=engine)
    wide = [torch.full((rows, 24 if columns > 8 else 8), 7.0, dtype=dtype, device="cuda:0") for _ in range(6)]
    x, o = ([w[:, :columns] for w in ws] for ws in (wide[:3], wide[3:]))
    for i, m in enumerate(x):
        m.copy_(_gradient(torch, shape, 40 + i, dtype))
    x[2], o[2] = x[2].t(), o[2].t()
    before = [w.clone() for w in wide]
    torch.cuda.synchronize()
    plan.orthogonalize(x, o)
    engine.synchronize()
    for a, b in zip(x, o):
        want, bound = _exact(a.double(), QUINTIC)
        _close(b, want, bound, _unit(ns_mode, a.shape), dtype)
    v = [torch.zeros_like(m) for m in x]
    plan.muon_step(o, x, v, lr=0.1)
    engine.synchronize()
    for w, b in zip(wide, before):
        assert torch.equal(w[:, columns:], b[:, columns:])
    assert all(torch.equal(w, b) for w, b in zip(wide[:3], before[:3]))


@gpu
def test_producers_and_consumers_on_other_streams(engine):
    """Inputs made on one stream, outputs read on another, ordered by events against the engine's stream."""
    import torch
    import volta_b200 as vb
    shapes = [(60, 500), (256, 300)]
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, engine=engine)
    xs = [torch.empty(s, device="cuda:0") for s in shapes]
    outs = [torch.empty(s, device="cuda:0") for s in shapes]
    tx, to = plan.matrices(xs), plan.matrices(outs)
    mine, producer, consumer = torch.cuda.ExternalStream(engine.stream), torch.cuda.Stream(), torch.cuda.Stream()
    kept = []
    torch.cuda.synchronize()
    for seed in range(6):
        with torch.cuda.stream(producer):
            producer.wait_stream(mine)
            for i, x in enumerate(xs):
                x.copy_(_gradient(torch, shapes[i], 100 * seed + i, torch.float32))
        mine.wait_stream(producer)
        mine.wait_stream(consumer)
        plan.orthogonalize(tx, to)
        consumer.wait_stream(mine)
        with torch.cuda.stream(consumer):
            kept.append([o.clone() for o in outs])
    torch.cuda.synchronize()
    for seed in range(6):
        for i, s in enumerate(shapes):
            want, bound = _exact(_gradient(torch, s, 100 * seed + i, torch.float32).double(), QUINTIC)
            _close(kept[seed][i], want, bound, _unit(vb.VB_NS_F16, s), torch.float32)


@gpu
def test_two_engines_at_once():
    """Plans of two engines, each with launches that want the whole device, enqueued without waiting."""
    import torch
    import volta_b200 as vb
    shapes = [(1024, 1024)] * 3 + [(64, 700)] * 5 + [(300, 1500)]
    engines = [vb.Engine(0), vb.Engine(0)]
    plans = [vb.NewtonSchulzPlan(shapes, QUINTIC, engine=e) for e in engines]
    xs = [_gradient(torch, s, 3 + i, torch.bfloat16) for i, s in enumerate(shapes)]
    outs = [[torch.empty_like(x) for x in xs] for _ in plans]
    alone = [torch.empty_like(x) for x in xs]
    torch.cuda.synchronize()
    plans[0].orthogonalize(xs, alone)
    engines[0].synchronize()
    tables = [(p.matrices(xs), p.matrices(o)) for p, o in zip(plans, outs)]
    for _ in range(5):
        for p, t in zip(plans, tables):
            p.orthogonalize(*t)
    for e in engines:
        e.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, alone))
    for p in plans:
        p.close()
    for e in engines:
        e.close()


@gpu
def test_engine_gone_and_workspace_refused():
    import torch
    import volta_b200 as vb
    eng = vb.Engine(0)
    with pytest.raises(vb.VoltaB200Error, match="workspace"):
        vb.NewtonSchulzPlan([(65536, 65536)] * 4, QUINTIC[:2], engine=eng)  # 240 GB
    plan = vb.NewtonSchulzPlan([(70, 80)], QUINTIC, engine=eng)
    x, o = torch.ones(70, 80, device="cuda:0"), torch.zeros(70, 80, device="cuda:0")
    plan.orthogonalize([x], [o])
    eng.synchronize()
    assert o.abs().max().item() > 0
    eng.close()
    with pytest.raises(vb.VoltaB200Error, match="destroyed"):
        plan.orthogonalize([x], [o])
    plan.close()
    with pytest.raises(vb.VoltaB200Error, match="null"):
        plan.orthogonalize([x], [o])


@gpu
@pytest.mark.parametrize("shapes", [[(300, 400)], [(50, 400)], [(50, 400), (300, 400)]])
def test_a_wait_that_runs_out_is_reported_and_stores_nothing(shapes):
    import torch
    import volta_b200 as vb
    from volta_b200 import _lib
    eng = vb.Engine(0)
    plan = vb.NewtonSchulzPlan(shapes, QUINTIC, engine=eng)
    xs = [_gradient(torch, s, 1, torch.float32) for s in shapes]
    outs = [torch.full_like(x, 3.0) for x in xs]
    torch.cuda.synchronize()
    _lib.call("vb_debug_ns_plan_withhold_loads", plan._h, 2000)
    plan.orthogonalize(xs, outs)
    with pytest.raises(vb.VoltaB200Error) as e:
        eng.synchronize()
    assert e.value.status == 4
    if len(shapes) == 1:  # of two launches side by side only the first one's waits run out
        assert (outs[0] == 3.0).all()
    with pytest.raises(vb.VoltaB200Error) as e:
        plan.orthogonalize(xs, outs)
    assert e.value.status == 4
    plan.close()
    fresh = vb.NewtonSchulzPlan(shapes, QUINTIC, engine=eng)  # the engine stays usable
    fresh.orthogonalize(xs, outs)
    eng.synchronize()
    assert not any((o == 3.0).any() for o in outs)
    fresh.close()
    eng.close()
