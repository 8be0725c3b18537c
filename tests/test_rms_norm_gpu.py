"""Root-mean-square norm (with the residual's addition, and with an 8-bit result) and its gradient against 64-bit numpy.

Tolerances.  u is the wide type's half step, ut the value type's.  A sum of C terms is formed in chains: a thread adds
its own terms (at most 32 in registers, C / 512 packets of up to 8 in the form for long rows), then 5 steps within a
warp and at most 32 across warps, so it is off by at most `chain` = C / 64 + 80 steps of the sum of the magnitudes.  The
expectation starts from the stored sum s and, for gradients, from the stored rstd: they are checked by themselves."""
import ctypes as C

import numpy as np
import pytest
import torch

from daphne_b200 import lib as names
from daphne_b200.lib import Db2Error, check, lib
from tests.seq_util import ALL, TYPES, Mat, assert_within, half_step, scratch, smallest, stream, wide

gpu = pytest.mark.gpu
EPS = 1e-5

SHAPES = [  # rows, cols, pad, shift
    (1, 1, 0, 0), (3, 7, 0, 0), (5, 64, 0, 0), (300, 33, 0, 0), (200, 129, 7, 0), (170, 333, 0, 1), (64, 1000, 24, 16),
    (1000, 512, 0, 0), (9, 4096, 0, 0), (300, 4100, 4, 8), (4, 9001, 0, 0), (160, 8200, 0, 8), (2, 16500, 12, 0),
    (3, 40000, 0, 0), (150, 33000, 0, 8), (40003, 8, 0, 0),
    (150, 12288, 0, 0), (4, 20480, 0, 0), (151, 640, 0, 0), (7000, 320, 0, 8), (6001, 24, 0, 0),
    (300, 130, 0, 0), (160, 2050, 2, 2), (3, 9002, 0, 0), (151, 5002, 0, 6),  # pairs
]


def _chain(cols):
    return cols / 64 + 80


def _forward(tname, rows, cols, pad, shift, residual=True, weight=True, group=None, seed=0, x=None, eps=EPS, rstd=True):
    t, code = TYPES[tname]
    rng = np.random.default_rng(seed + rows + cols)
    X = Mat(rng.standard_normal((rows, cols)) * 2 if x is None else x, t, pad, shift)
    R = Mat(rng.standard_normal((rows, cols)) * 3 + 0.3, t, pad, shift) if residual else None
    W = Mat(rng.standard_normal((1, cols)) * 0.3 + 1, t, 0, shift) if weight else None
    S = Mat.empty(rows, cols, t, pad, shift) if residual else None
    Y = Mat.empty(rows, cols, t if group is None else torch.float8_e4m3fn, pad, shift) if group is None else \
        Mat(torch.zeros(rows, cols), torch.uint8, pad, shift)
    V = Mat.empty(rows, 1, wide(t)) if rstd else None
    args = (code, X.ptr, rows, cols, X.ld, R.ptr if R else None, R.ld if R else 0, W.ptr if W else None, eps,
            S.ptr if S else None, S.ld if S else 0, *Y.at)
    if group is None:
        check(lib.db2k_rms_norm(*args, V.ptr if V else None, stream()))
        Q = None
    else:
        Q = Mat.empty(rows, -(-cols // group) if group else 1, torch.float32, 2)
        check(lib.db2k_rms_norm_q8(*args, *Q.at, group, V.ptr if V else None, stream()))
    return X, R, W, S, Y, V, Q


def _check_front(tname, X, R, S, V, eps=EPS):
    """The stored sum and rstd; returns s in 64 bits and the relative error that rstd may have."""
    t = TYPES[tname][0]
    u, ut = half_step(wide(t)), half_step(t)
    s = X.f64()
    if R is not None:
        exact = s + R.f64()
        s = S.f64()
        # one rounding to the wide type and one to the value type
        assert_within(s, exact, np.abs(exact) * (ut + 2 * u) + smallest(t), "sum")
        assert S.guards_intact()
    rel = (_chain(s.shape[1]) / 2 + 4) * u
    if V is not None:
        exp = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
        assert_within(V.f64(), exp, exp * rel, "rstd")
        assert V.guards_intact()
    return s, rel


@gpu
@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("rows,cols,pad,shift", SHAPES)
def test_norm(tname, rows, cols, pad, shift):
    t = TYPES[tname][0]
    u, ut = half_step(wide(t)), half_step(t)
    for residual, weight in ((True, True), (False, False)):
        X, R, W, S, Y, V, _ = _forward(tname, rows, cols, pad, shift, residual, weight)
        s, rel = _check_front(tname, X, R, S, V)
        exp = s / np.sqrt((s * s).mean(1, keepdims=True) + EPS) * (W.f64() if W else 1.0)
        assert_within(Y.f64(), exp, np.abs(exp) * (rel + 3 * u + ut) + smallest(t), "rmsNorm")
        assert Y.guards_intact() and X.guards_intact()


def _e4m3(Y):
    return Y.view.view(torch.float8_e4m3fn).double().cpu().numpy()


@gpu
@pytest.mark.parametrize("tname", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [0, 16, 32, 128, 256, 512])
@pytest.mark.parametrize("rows,cols,pad,shift", SHAPES)
def test_norm_in_eight_bits(tname, group, rows, cols, pad, shift):
    t = TYPES[tname][0]
    u = half_step(wide(t))
    X, R, W, S, Y, V, Q = _forward(tname, rows, cols, pad, shift, True, True, group)
    s, rel = _check_front(tname, X, R, S, V)
    y = s / np.sqrt((s * s).mean(1, keepdims=True) + EPS) * W.f64()
    width = group or cols
    n = -(-cols // width)
    full = np.zeros((rows, n * width))
    full[:, :cols] = np.abs(y)
    scale = full.reshape(rows, n, width).max(2) / 448
    assert_within(Q.f64(), scale, scale * (rel + 4 * u), "scales")
    assert Q.guards_intact()
    per = np.repeat(Q.f64(), width, 1)[:, :cols]
    # the quotient is off by a few u, its rounding by half a step (2^-4), or half a subnormal's distance (2^-10)
    assert_within(_e4m3(Y) * per, y, np.abs(y) * (2.0 ** -4 + rel + 6 * u) + per * 2.0 ** -10, "rmsNormQ8")
    # where no border is near, the value is the nearest one
    q = torch.as_tensor(y / per)
    near = np.abs(q.numpy()) * (rel + 8 * u)
    lo, hi = (q - torch.as_tensor(near)).float().to(torch.float8_e4m3fn), (q + torch.as_tensor(near)).float().to(torch.float8_e4m3fn)
    sure = (lo.view(torch.uint8) == hi.view(torch.uint8)).numpy()
    assert sure.mean() > 0.99 or sure.size < 1000
    assert np.array_equal(_e4m3(Y)[sure], lo.double().numpy()[sure])
    assert bool((Y.buf[Y.shift:Y.shift + rows * Y.ld].view(rows, Y.ld)[:, cols:] == 77).all())


def _backward(tname, rows, cols, pad, shift, dsum=True, weight=True, seed=1):
    t, code = TYPES[tname]
    X, R, W, S, Y, V, _ = _forward(tname, rows, cols, pad, shift, True, weight)
    rng = np.random.default_rng(seed + rows + cols)
    G = Mat(rng.standard_normal((rows, cols)), t, pad, shift)
    D = Mat(rng.standard_normal((rows, cols)), t, pad, shift) if dsum else None
    O, DW = Mat.empty(rows, cols, t, pad, shift), Mat.empty(1, cols, wide(t))
    n = lib.db2k_rms_norm_grad_scratch_bytes(code, rows, cols)
    sc = scratch(n)

    def call():
        check(lib.db2k_rms_norm_grad(code, *G.at, rows, cols, *S.at, W.ptr if W else None, V.ptr, D.ptr if D else None,
                                     D.ld if D else 0, *O.at, DW.ptr, sc.data_ptr(), n, stream()))
    call()
    return G, S, W, V, D, O, DW, call


def _expect_grad(G, S, W, V, D):
    g, s, r = G.f64(), S.f64(), V.f64()
    t = g * (W.f64() if W else 1.0)
    dot = (t * s).mean(1, keepdims=True)
    dx = r * (t - s * r * r * dot) + (D.f64() if D else 0.0)
    mag = r * (np.abs(t) + np.abs(s) * r * r * np.abs(t * s).mean(1, keepdims=True)) + (np.abs(D.f64()) if D else 0.0)
    return dx, mag, (g * s * r).sum(0, keepdims=True), np.abs(g * s * r).sum(0, keepdims=True)


@gpu
@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("rows,cols,pad,shift", SHAPES)
def test_gradient(tname, rows, cols, pad, shift):
    t = TYPES[tname][0]
    u, ut = half_step(wide(t)), half_step(t)
    for dsum, weight in ((True, True), (False, False)):
        G, S, W, V, D, O, DW, call = _backward(tname, rows, cols, pad, shift, dsum, weight)
        dx, mag, dw, dwmag = _expect_grad(G, S, W, V, D)
        assert_within(O.f64(), dx, np.abs(dx) * ut + mag * (_chain(cols) + 10) * u + smallest(t), "dx")
        assert_within(DW.f64(), dw, dwmag * (rows + 4) * u + smallest(wide(t)), "dweight")
        assert O.guards_intact() and DW.guards_intact() and G.guards_intact()
        first, firstw = O.view.clone(), DW.view.clone()
        call()
        assert torch.equal(first, O.view) and torch.equal(firstw, DW.view), "the same bits in every run"


@gpu
def test_gradient_agrees_with_differences():
    rng = np.random.default_rng(8)
    rows, cols = 3, 6
    x, r, w, c = (rng.standard_normal(s) for s in ((rows, cols), (rows, cols), (1, cols), (rows, cols)))
    e = rng.standard_normal((rows, cols))

    def f(x, w):  # a function of both results
        s = x + r
        y = s / np.sqrt((s * s).mean(1, keepdims=True) + EPS) * w
        return float((y * c).sum() + (s * e).sum())
    code, t = names.F64, torch.float64
    X, R, W = Mat(x, t), Mat(r, t), Mat(w, t)
    S, Y, V = Mat.empty(rows, cols, t), Mat.empty(rows, cols, t), Mat.empty(rows, 1, t)
    check(lib.db2k_rms_norm(code, X.ptr, rows, cols, cols, *R.at, W.ptr, EPS, *S.at, *Y.at, V.ptr, stream()))
    assert abs(float((Y.f64() * c).sum() + (S.f64() * e).sum()) - f(x, w)) < 1e-12
    G, D, O, DW = Mat(c, t), Mat(e, t), Mat.empty(rows, cols, t), Mat.empty(1, cols, t)
    n = lib.db2k_rms_norm_grad_scratch_bytes(code, rows, cols)
    check(lib.db2k_rms_norm_grad(code, *G.at, rows, cols, *S.at, W.ptr, V.ptr, *D.at, *O.at, DW.ptr, scratch(n).data_ptr(),
                                 n, stream()))
    h = 1e-5  # third derivatives are of the order of 10: the differences are good to 10 h^2 + 1e-15 / h
    for got, arg in ((O.f64(), 0), (DW.f64(), 1)):
        for i in np.ndindex(got.shape):
            d = [np.zeros_like(x), np.zeros_like(w)]
            d[arg][i] = h
            diff = (f(x + d[0], w + d[1]) - f(x - d[0], w - d[1])) / (2 * h)
            assert abs(diff - got[i]) < 1e-7


@gpu
@pytest.mark.parametrize("tname", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [96, 4096, 40000])
def test_results_in_the_place_of_operands(tname, cols):
    """sum over x or residual, result over x, dx over grad, sum or dsum: the same bits as with matrices of their own."""
    t, code = TYPES[tname]
    rows = 20
    X, R, W, S, Y, V, _ = _forward(tname, rows, cols, 0, 0)
    x0, r0 = X.buf.clone(), R.buf.clone()
    for sum_at, res_at in ((X, R), (R, X), (X, Y), (R, Y), (None, X), (None, R)):
        X.buf.copy_(x0)
        R.buf.copy_(r0)
        check(lib.db2k_rms_norm(code, X.ptr, rows, cols, X.ld, *R.at, W.ptr, EPS, *(sum_at.at if sum_at else (None, 0)),
                                *res_at.at, V.ptr, stream()))
        exp = Mat.empty(rows, cols, t)
        rst = Mat.empty(rows, 1, wide(t))
        X2, R2 = Mat(torch.zeros(rows, cols), t), Mat(torch.zeros(rows, cols), t)
        X2.buf.copy_(x0)
        R2.buf.copy_(r0)
        check(lib.db2k_rms_norm(code, X2.ptr, rows, cols, X2.ld, *R2.at, W.ptr, EPS, *S.at, *exp.at, rst.ptr, stream()))
        assert torch.equal(res_at.view, exp.view) and torch.equal(V.view, rst.view)
        if sum_at:
            assert torch.equal(sum_at.view, S.view)
    G, S, W, V, D, O, DW, call = _backward(tname, rows, cols, 0, 0)
    exp, expw = O.view.clone(), DW.view.clone()
    n = lib.db2k_rms_norm_grad_scratch_bytes(code, rows, cols)
    sc = scratch(n)
    keep = [m.buf.clone() for m in (G, S, D)]
    for target in (G, S, D):
        for m, b in zip((G, S, D), keep):
            m.buf.copy_(b)
        check(lib.db2k_rms_norm_grad(code, *G.at, rows, cols, *S.at, W.ptr, V.ptr, *D.at, *target.at, DW.ptr,
                                     sc.data_ptr(), n, stream()))
        assert torch.equal(target.view, exp) and torch.equal(DW.view, expw)


@gpu
@pytest.mark.parametrize("cols", [40, 3000, 40000])
def test_rows_of_zeros_infinities_and_nan_stay_by_themselves(cols):
    x = np.random.default_rng(2).standard_normal((5, cols))
    x[1] = 0
    x[2, 3] = np.inf
    x[3, 5] = np.nan
    for tname in ALL:
        X, _, W, _, Y, V, _ = _forward(tname, 5, cols, 0, 0, False, True, x=x)
        y, r = Y.f64(), V.f64()[:, 0]
        assert np.isfinite(y[[0, 1, 4]]).all() and not y[1].any() and abs(r[1] - EPS ** -0.5) < 1e-3
        assert r[2] == 0 and np.isnan(y[2, 3]) and not y[2, np.arange(cols) != 3].any()
        assert np.isnan(y[3]).all() and np.isnan(r[3])
    X, _, W, _, Y, V, Q = _forward("bf16", 5, cols, 0, 0, False, True, group=32, x=x)
    q, sc = _e4m3(Y), Q.f64()
    assert (sc[1] == 1).all() and not q[1].any() and np.isfinite(q[[0, 4]]).all()
    assert np.isnan(sc[3]).all() and np.isnan(q[3]).all() and np.isnan(sc[2, 0])
    # the smallest numbers: scales that stay normal, values that stay finite
    tiny = np.zeros((1, cols))
    tiny[0, 0] = 1e-38
    _, _, _, _, Y, _, Q = _forward("f32", 1, cols, 0, 0, False, False, group=0, x=tiny, eps=1.0)
    assert Q.f64()[0, 0] >= 1.17e-38 and np.isfinite(_e4m3(Y)).all()


@gpu
def test_optional_results_and_a_captured_call():
    t, code = TYPES["bf16"]
    X, R, W, S, Y, V, _ = _forward("bf16", 50, 640, 0, 0)
    Y2 = Mat.empty(50, 640, t)
    check(lib.db2k_rms_norm(code, X.ptr, 50, 640, 640, *R.at, W.ptr, EPS, None, 0, *Y2.at, None, stream()))
    assert torch.equal(Y.view, Y2.view)
    G, S, W, V, D, O, DW, call = _backward("bf16", 50, 640, 0, 0)
    O2 = Mat.empty(50, 640, t)
    check(lib.db2k_rms_norm_grad(code, *G.at, 50, 640, *S.at, W.ptr, V.ptr, *D.at, *O2.at, None, None, 0, stream()))
    assert torch.equal(O.view, O2.view)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    G.view.normal_()
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    a, b = O.view.clone(), DW.view.clone()
    call()
    assert torch.equal(a, O.view) and torch.equal(b, DW.view)


@gpu
def test_on_handles(ctx):
    import daphne_b200.kernels as k
    rng = np.random.default_rng(9)
    x, r, w, g = (rng.standard_normal(s) for s in ((300, 70), (300, 70), (1, 70), (300, 70)))
    X, R, W, G = (k.DenseMatrix.from_numpy(ctx, a) for a in (x, r, w, g))
    y, s, rstd = k.rmsNorm(X, W, EPS, residual=R)
    s64 = x + r
    exp = s64 / np.sqrt((s64 * s64).mean(1, keepdims=True) + EPS)
    np.testing.assert_allclose(y.to_numpy(), exp * w, rtol=1e-13, atol=0)
    assert np.array_equal(s.to_numpy(), s64)
    dx, dw = k.rmsNormGrad(G, s, rstd, W, dsum=G)
    rs = rstd.to_numpy()
    t = g * w
    e = rs * (t - s64 * rs * rs * (t * s64).mean(1, keepdims=True)) + g
    np.testing.assert_allclose(dx.to_numpy(), e, rtol=0, atol=1e-13)
    np.testing.assert_allclose(dw.to_numpy(), (g * s64 * rs).sum(0, keepdims=True), rtol=0, atol=1e-11)
    # column views (odd offsets and a leading dimension of their own), deferred chains, no weight
    Z = k.ewBinaryObjSca(k.BinaryOpCode.MUL, X, 2.0)
    y2, s2, _ = k.rmsNorm(Z, eps=EPS)
    assert s2 is Z
    z = 2 * x
    np.testing.assert_allclose(y2.to_numpy(), z / np.sqrt((z * z).mean(1, keepdims=True) + EPS), rtol=1e-13, atol=0)
    v = x[:, 3:40]
    y3, _, _ = k.rmsNorm(k.sliceCol(X, 3, 40), k.sliceCol(W, 3, 40), EPS)
    np.testing.assert_allclose(y3.to_numpy(), v / np.sqrt((v * v).mean(1, keepdims=True) + EPS) * w[:, 3:40], rtol=1e-13)
    X32, W32 = k.castObj(X, np.float32), k.castObj(W, np.float32)
    q, sc, _, _ = k.rmsNormQ8(X32, W32, EPS, group=16)
    assert sc.shape == (300, 5)
    y32 = k.rmsNorm(X32, W32, EPS)[0].to_numpy()
    deq = k.castObj(q, np.float32).to_numpy() * np.repeat(sc.to_numpy(), 16, 1)[:, :70]
    assert (np.abs(deq - y32) <= np.abs(y32) * (2.0 ** -4 + 1e-6) + np.repeat(sc.to_numpy(), 16, 1)[:, :70] * 2.0 ** -10).all()
    for call, msg in ((lambda: k.rmsNorm(X, W, -1.0), "eps must not be negative"),
                      (lambda: k.rmsNorm(X, W, float("nan")), "eps must not be negative"),
                      (lambda: k.rmsNorm(X, X), "weight must be a row matrix"),
                      (lambda: k.rmsNorm(X, W32), "weight must be a row matrix"),
                      (lambda: k.rmsNorm(X, residual=X32), "residual must have"),
                      (lambda: k.rmsNormQ8(X, W), "unsupported value type"),
                      (lambda: k.rmsNormQ8(X32, W32, group=48), "groups of 16"),
                      (lambda: k.rmsNorm(k.castObj(X, np.int64)), "unsupported value type"),
                      (lambda: k.rmsNormGrad(G, s, k.castObj(rstd, np.float32), W), "rstd must be"),
                      (lambda: k.rmsNormGrad(G, k.sliceRow(s, 0, 10), rstd, W), "sum must have")):
        with pytest.raises(Db2Error, match=msg):
            call()
    # a result that names its own operand gets a new buffer: the operand's other handles keep their values
    h, keep = k.castObj(X, np.float64), x.copy()
    chain = k.ewBinaryObjSca(k.BinaryOpCode.ADD, h, 0.0)
    check(lib.db2_rmsNorm(ctx.handle, C.byref(h._h), None, None, h.handle, None, None, EPS))
    np.testing.assert_allclose(h.to_numpy(), x / np.sqrt((x * x).mean(1, keepdims=True) + EPS), rtol=1e-13)
    assert np.array_equal(chain.to_numpy(), keep)


def test_refusals():
    buf = (C.c_char * 8192)()
    p = C.addressof(buf)
    p += -p % 16

    def refused(code, call):
        with pytest.raises(Db2Error) as e:
            check(call())
        assert e.value.code == code, e.value
    base = dict(dt=names.BF16, x=p, rows=4, cols=32, ld=32, r=p, rld=32, w=p, eps=1e-6, s=p, sld=32, y=p, yld=32, q=p, qld=2,
                group=16, v=p)

    def norm(**kw):
        a = {**base, **kw}
        return lib.db2k_rms_norm(a["dt"], a["x"], a["rows"], a["cols"], a["ld"], a["r"], a["rld"], a["w"], a["eps"], a["s"],
                                 a["sld"], a["y"], a["yld"], a["v"], None)

    def q8(**kw):
        a = {**base, **kw}
        return lib.db2k_rms_norm_q8(a["dt"], a["x"], a["rows"], a["cols"], a["ld"], a["r"], a["rld"], a["w"], a["eps"],
                                    a["s"], a["sld"], a["y"], a["yld"], a["q"], a["qld"], a["group"], a["v"], None)
    for f in (norm, q8):
        for dt in (names.I64, names.F8E4M3, 50):
            refused(4, lambda: f(dt=dt))
        for kw in (dict(rows=-1), dict(cols=-1), dict(cols=0), dict(x=None), dict(y=None), dict(ld=31), dict(rld=31),
                   dict(sld=31), dict(yld=31), dict(eps=-1.0), dict(eps=float("nan"))):
            refused(1, lambda: f(**kw))
        assert f(rows=0, x=None) == 0
    refused(4, lambda: q8(dt=names.F64))
    for kw in (dict(group=8), dict(group=48), dict(group=1024), dict(group=-16), dict(q=None), dict(qld=1)):
        refused(1, lambda: q8(**kw))
    g = dict(dt=names.F32, g=p, gld=32, rows=4, cols=32, s=p, sld=32, w=p, v=p, d=p, dld=32, dx=p, xld=32, dw=p, sc=p, sb=8192)

    def grad(**kw):
        a = {**g, **kw}
        return lib.db2k_rms_norm_grad(a["dt"], a["g"], a["gld"], a["rows"], a["cols"], a["s"], a["sld"], a["w"], a["v"],
                                      a["d"], a["dld"], a["dx"], a["xld"], a["dw"], a["sc"], a["sb"], None)
    refused(4, lambda: grad(dt=names.U8))
    for kw in (dict(rows=-1), dict(g=None), dict(s=None), dict(v=None), dict(dx=None), dict(gld=31), dict(sld=31),
               dict(dld=31), dict(xld=31), dict(sc=None), dict(sc=p + 4), dict(sb=8)):
        refused(1, lambda: grad(**kw))
    assert grad(cols=0) == 0
    assert lib.db2k_rms_norm_grad_scratch_bytes(names.F32, 0, 32) == 0
