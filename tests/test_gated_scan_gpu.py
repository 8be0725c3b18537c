"""Gated linear recurrence over packed sequences, its gradient and its single-row step against plain 64-bit loops.

Tolerances.  u is the wide type's half step, ut the value type's.  With M[t] = |f[t]| M[t-1] + |u[t]| (the recurrence of the
magnitudes) every rounding on the way from an input to h[t] -- of a sum, of a product of gates, of a gate -- is at most k
steps of what passes through row s, so the error obeys E[t] = |f[t]| E[t-1] + k u M[t].  k = 4 for the sums and products;
a sigmoid in single precision adds what the fast exponential (2 + 1.16 |g| units in the last place) and the division
(2 units) may cost, a unit being two half steps: 2 (6 + 1.2 max|g|)."""
import ctypes as C

import numpy as np
import pytest
import torch

from daphne_b200 import lib as names
from daphne_b200.lib import Db2Error, check, lib
from tests.seq_util import ALL, GUARD, TYPES, Mat, assert_within, half_step, scratch, smallest, stream, wide

gpu = pytest.mark.gpu
DECAY, SIGMOID = names.GATE_DECAY, names.GATE_SIGMOID

CASES = [  # rows, cols, offsets (a number: that many equally long sequences), pad, shift
    (1, 1, 1, 0, 0), (5, 3, 1, 0, 0), (63, 64, 1, 0, 0), (64, 65, 1, 1, 1), (65, 40, 1, 0, 0), (129, 130, 3, 2, 2),
    (1000, 70, 1, 0, 0), (2400, 33, 8, 3, 0), (60, 200, 60, 0, 8), (700, 96, [0, 1, 1, 64, 130, 131, 500, 500, 650], 0, 0),
    (300, 38, [7, 7, 100, 290], 10, 2), (40, 5, [3, 3], 0, 0), (900, 2, 2, 0, 0),
    (20000, 5, 1, 0, 0), (9001, 34, [0, 1500, 1501, 9000], 0, 0),  # cut into blocks
    (4, 20000, 2, 0, 0), (0, 6, 3, 0, 0),
]


def _offsets(rows, off):
    if isinstance(off, int):
        return np.arange(off + 1) * (rows // off), None
    return np.array(off), torch.tensor(off, dtype=torch.int64, device="cuda")


def _inputs(tname, gate, rows, cols, off, pad=0, shift=0, seed=0, state=True):
    t = TYPES[tname][0]
    rng = np.random.default_rng(seed + rows * 7 + cols)
    g = rng.standard_normal((rows, cols)) * 2 + 1 if gate == SIGMOID else 1 - 0.4 * rng.random((rows, cols)) ** 3
    if rows and gate == DECAY:
        g[rng.random((rows, cols)) < 0.05] *= -1
        g[rng.random((rows, cols)) < 0.02] = 0
        g[rng.random((rows, cols)) < 0.05] = 1
    seqs = len(off) - 1
    G, X = Mat(g, t, pad, shift), Mat(rng.standard_normal((rows, cols)), t, pad, shift)
    H0 = Mat(rng.standard_normal((seqs, cols)), wide(t), 1) if state else None
    return G, X, H0


def _at(m):
    return m.at if m is not None else (None, 0)


def _scan(tname, gate, G, X, seqs, dev_off, H0, H=None, last=True):
    t, code = TYPES[tname]
    H = H or Mat.empty(G.rows, G.cols, t, G.ld - G.cols, G.shift)
    L = Mat.empty(seqs, G.cols, wide(t), 2) if last else None
    n = lib.db2k_gated_scan_scratch_bytes(code, G.rows, G.cols, seqs)
    s = scratch(n)
    check(lib.db2k_gated_scan(code, gate, *G.at, *X.at, G.rows, G.cols, None if dev_off is None else dev_off.data_ptr(), seqs,
                              *_at(H0), *H.at, *_at(L), s.data_ptr(), n, stream()))
    return H, L


def _gates(gate, g, x):
    if gate == DECAY:
        return g, np.ones_like(g), x
    with np.errstate(over="ignore"):
        f, o = 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))
    return f, o, o * x


def _k(tname, gate, g):
    return 4 + (2 * (6 + 1.2 * np.abs(g).max(initial=0)) if gate == SIGMOID else 0)


def _expect(tname, gate, G, X, off, H0):
    """h, last, and how far each may be off before the rounding to the value type"""
    g, x = G.f64(), X.f64()
    u, k = half_step(wide(TYPES[tname][0])), _k(tname, gate, g)
    f, _, b = _gates(gate, g, x)
    h, err = np.full(g.shape, GUARD), np.zeros(g.shape)
    seqs = len(off) - 1
    last, lerr = np.zeros((seqs, g.shape[1])), np.zeros((seqs, g.shape[1]))
    h0 = H0.f64() if H0 is not None else np.zeros_like(last)
    for s in range(seqs):
        v, m, e = h0[s], np.abs(h0[s]), 0
        for r in range(off[s], off[s + 1]):
            v, m = f[r] * v + b[r], np.abs(f[r]) * m + np.abs(b[r])
            e = np.abs(f[r]) * e + k * u * m
            h[r], err[r] = v, e
        last[s], lerr[s] = v, e
    return h, err, last, lerr


@gpu
@pytest.mark.parametrize("gate", [DECAY, SIGMOID])
@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("rows,cols,off,pad,shift", CASES)
def test_scan(tname, gate, rows, cols, off, pad, shift):
    t = TYPES[tname][0]
    off, dev = _offsets(rows, off)
    for state in (True, False):
        G, X, H0 = _inputs(tname, gate, rows, cols, off, pad, shift, state=state)
        H, L = _scan(tname, gate, G, X, len(off) - 1, dev, H0)
        h, err, last, lerr = _expect(tname, gate, G, X, off, H0)
        assert_within(H.f64(), h, err + np.abs(h) * half_step(t) + smallest(t), "h")
        assert_within(L.f64(), last, lerr + smallest(wide(t)), "last")
        outside = np.ones(rows, dtype=bool)
        outside[off[0]:off[-1]] = False
        assert (H.f64()[outside] == GUARD).all(), "rows of no sequence stay"
        assert H.guards_intact() and L.guards_intact() and G.guards_intact()


def _grad(tname, gate, G, X, H, D, seqs, dev_off, H0, DL):
    t, code = TYPES[tname]
    new = lambda: Mat.empty(G.rows, G.cols, t, G.ld - G.cols, G.shift)  # noqa: E731
    DG, DX, DH0 = new(), new(), Mat.empty(seqs, G.cols, wide(t), 1)
    n = lib.db2k_gated_scan_scratch_bytes(code, G.rows, G.cols, seqs)
    s = scratch(n)
    check(lib.db2k_gated_scan_grad(code, gate, *G.at, *_at(X if gate == SIGMOID else None), *H.at, *D.at, G.rows, G.cols,
                                   None if dev_off is None else dev_off.data_ptr(), seqs, *_at(H0), *_at(DL), *DG.at,
                                   *DX.at, *DH0.at, s.data_ptr(), n, stream()))
    return DG, DX, DH0


@gpu
@pytest.mark.parametrize("gate", [DECAY, SIGMOID])
@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("rows,cols,off,pad,shift", CASES)
def test_gradient(tname, gate, rows, cols, off, pad, shift):
    t = TYPES[tname][0]
    ut, u = half_step(t), half_step(wide(t))
    off, dev = _offsets(rows, off)
    seqs = len(off) - 1
    for state in (True, False):
        G, X, H0 = _inputs(tname, gate, rows, cols, off, pad, shift, state=state)
        H, _ = _scan(tname, gate, G, X, seqs, dev, H0)
        rng = np.random.default_rng(99)
        D = Mat(rng.standard_normal((rows, cols)), t, pad, shift)
        DL = Mat(rng.standard_normal((seqs, cols)), wide(t), 3) if state else None
        DG, DX, DH0 = _grad(tname, gate, G, X, H, D, seqs, dev, H0, DL)
        g, x, h, d = G.f64(), X.f64(), H.f64(), D.f64()
        k = _k(tname, gate, g)
        f, o, _ = _gates(gate, g, x)
        dg, dx = np.full(g.shape, GUARD), np.full(g.shape, GUARD)
        bg, bx = np.zeros(g.shape), np.zeros(g.shape)
        h0 = H0.f64() if state else np.zeros((seqs, cols))
        c0, b0 = np.zeros((seqs, cols)), np.zeros((seqs, cols))
        for s in range(seqs):
            c = DL.f64()[s] if state else np.zeros(cols)
            m, e = np.abs(c), 0 * c
            for r in range(off[s + 1] - 1, off[s] - 1, -1):
                delta, m = d[r] + c, np.abs(d[r]) + m
                e = e + k * u * m
                above = h[r - 1] if r > off[s] else h0[s]
                if gate == SIGMOID:
                    w = f[r] * o[r]
                    dg[r], dx[r] = delta * (above - x[r]) * w, delta * o[r]
                    bg[r] = (e * np.abs(above - x[r]) + np.abs(delta) * (np.abs(above) + np.abs(x[r])) * 3 * k * u) * w
                    bx[r] = (e + np.abs(delta) * k * u) * o[r]
                else:
                    dg[r], dx[r] = delta * above, delta
                    bg[r], bx[r] = (e + np.abs(delta) * 2 * u) * np.abs(above), e
                c, m, e = f[r] * delta, np.abs(f[r]) * m, np.abs(f[r]) * e
            c0[s], b0[s] = c, e + k * u * m
        assert_within(DG.f64(), dg, bg + np.abs(dg) * ut + smallest(t), "dg")
        assert_within(DX.f64(), dx, bx + np.abs(dx) * ut + smallest(t), "dx")
        assert_within(DH0.f64(), c0, b0 + smallest(wide(t)), "dh0")
        assert DG.guards_intact() and DX.guards_intact() and DH0.guards_intact()
        again = _grad(tname, gate, G, X, H, D, seqs, dev, H0, DL)
        assert all(torch.equal(a.view, b.view) for a, b in zip(again, (DG, DX, DH0))), "the same bits in every run"


@gpu
@pytest.mark.parametrize("gate", [DECAY, SIGMOID])
def test_gradient_agrees_with_differences(gate):
    off, dev = _offsets(9, [0, 4, 4, 8])
    G, X, H0 = _inputs("f64", gate, 9, 3, off)
    rng = np.random.default_rng(5)
    w, wl = rng.standard_normal((9, 3)), rng.standard_normal((3, 3))
    w[8] = 0  # a row of no sequence

    def f(g, x, h0):
        H, L = _scan("f64", gate, Mat(g, torch.float64), Mat(x, torch.float64), 3, dev, Mat(h0, torch.float64))
        return float((H.f64() * w).sum() + (L.f64() * wl).sum())
    base = [G.f64(), X.f64(), H0.f64()]
    H, _ = _scan("f64", gate, G, X, 3, dev, H0)
    got = [m.f64() for m in _grad("f64", gate, G, X, H, Mat(w, torch.float64), 3, dev, H0, Mat(wl, torch.float64))]
    step = 1e-5  # differences of sums of about 40 values of up to 10: 1e-14 / step, and third derivatives times step^2
    for k in range(3):
        for i in np.ndindex(base[k].shape):
            if k < 2 and i[0] == 8:
                continue
            a, b = [v.copy() for v in base], [v.copy() for v in base]
            a[k][i] += step
            b[k][i] -= step
            assert abs((f(*a) - f(*b)) / (2 * step) - got[k][i]) < 1e-7


@gpu
@pytest.mark.parametrize("gate", [DECAY, SIGMOID])
@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("n,cols,pad,shift", [(1, 1, 0, 0), (3, 70, 2, 1), (64, 2048, 0, 0), (2, 7001, 0, 0), (70000, 3, 0, 0),
                                              (33, 256, 8, 8)])
def test_step(tname, gate, n, cols, pad, shift):
    t, code = TYPES[tname]
    off = np.arange(n + 1)
    G, X, H0 = _inputs(tname, gate, n, cols, off, pad, shift)
    N, H = Mat.empty(n, cols, wide(t), 3), Mat.empty(n, cols, t, pad, shift)
    check(lib.db2k_gated_step(code, gate, *G.at, *X.at, n, cols, *H0.at, *N.at, *H.at, stream()))
    g, x = G.f64(), X.f64()
    f, _, b = _gates(gate, g, x)
    v = f * H0.f64() + b
    err = _k(tname, gate, g) * half_step(wide(t)) * (np.abs(f * H0.f64()) + np.abs(b))
    assert_within(N.f64(), v, err + smallest(wide(t)), "state")
    assert_within(H.f64(), v, err + np.abs(v) * half_step(t) + smallest(t), "h")
    assert N.guards_intact() and H.guards_intact()
    # in place, without h, and as a scan over sequences of one row
    keep = N.view.clone()
    check(lib.db2k_gated_step(code, gate, *G.at, *X.at, n, cols, *H0.at, *H0.at, None, 0, stream()))
    assert torch.equal(H0.view, keep)


@gpu
def test_steps_and_chunks_continue_a_scan():
    """A sequence in one call, in two calls that hand on the state, and row by row: the same values up to rounding."""
    for gate in (DECAY, SIGMOID):
        off, _ = _offsets(200, 1)
        G, X, H0 = _inputs("f32", gate, 200, 50, off)
        H, L = _scan("f32", gate, G, X, 1, None, H0)
        cut = 77
        parts, state = [], H0
        for a, b in ((0, cut), (cut, 200)):
            h, state = _scan("f32", gate, Mat(G.view[a:b], torch.float32), Mat(X.view[a:b], torch.float32), 1, None, state)
            parts.append(h.f64())
        _, err, _, lerr = _expect("f32", gate, G, X, off, H0)
        assert_within(np.concatenate(parts), H.f64(), 2 * err + np.abs(H.f64()) * 2.0 ** -23, "two chunks")
        S = Mat(H0.view, torch.float32)
        for r in range(200):
            g, x = Mat(G.view[r:r + 1], torch.float32), Mat(X.view[r:r + 1], torch.float32)
            check(lib.db2k_gated_step(names.F32, gate, *g.at, *x.at, 1, 50, *S.at, *S.at, None, 0, stream()))
        assert_within(S.f64(), L.f64(), 2 * lerr, "row by row")


@gpu
@pytest.mark.parametrize("rows", [200, 20000])
def test_non_finite_values_stay_in_their_column_and_sequence(rows):
    off, dev = _offsets(rows, [0, rows // 2, rows])
    for tname in ALL:
        for gate in (DECAY, SIGMOID):
            G, X, H0 = _inputs(tname, gate, rows, 6, off)
            clean = _scan(tname, gate, G, X, 2, dev, H0)[0].f64()
            X.view[3, 1] = float("nan")
            X.view[5, 2] = float("inf")
            if gate == DECAY:  # neither a gate of zero nor an underflowing product makes a later row finite again
                G.view[:, 1:3] = 0.5
                clean[:, 1:3] = _scan(tname, gate, G, Mat(torch.where(X.view.isfinite(), X.view, 0), TYPES[tname][0]), 2, dev, H0)[0].f64()[:, 1:3]
            H, L = _scan(tname, gate, G, X, 2, dev, H0)
            got = H.f64()
            assert not np.isfinite(got[3:rows // 2, 1]).any() and not np.isfinite(got[5:rows // 2, 2]).any()
            bad = np.zeros(got.shape, dtype=bool)
            bad[3:rows // 2, 1] = bad[5:rows // 2, 2] = True
            assert np.array_equal(got[~bad], clean[~bad])
            assert np.isfinite(L.f64()[1]).all() and not np.isfinite(L.f64()[0, 1:3]).any()


@gpu
@pytest.mark.parametrize("rows", [200, 20000])
@pytest.mark.parametrize("row", [0, 3, 8, 31, 32, 64, 77])
def test_gates_that_are_not_finite(rows, row):
    """They reach all later rows of their column and sequence (earlier ones in the gradient), whatever the state is."""
    off, dev = _offsets(rows, [0, rows // 2, rows])
    for tname in ("f32", "f64", "bf16"):
        t = TYPES[tname][0]
        for bad in (float("nan"), float("inf")):
            g = np.full((rows, 5), 0.5)
            g[row, 1] = bad
            G, X = Mat(g, t), Mat(np.zeros((rows, 5)), t)
            H, L = _scan(tname, DECAY, G, X, 2, dev, None)  # a state of zero in front of it
            h = H.f64()
            assert not np.isfinite(h[row:rows // 2, 1]).any() and not np.isfinite(L.f64()[0, 1])
            keep = np.ones(h.shape, dtype=bool)
            keep[row:rows // 2, 1] = False
            assert not h[keep].any() and not L.f64()[1].any()
            D = Mat(np.ones((rows, 5)), t)
            clean = _scan(tname, DECAY, Mat(np.full((rows, 5), 0.5), t), X, 2, dev, None)[0]
            DG, DX, DH0 = _grad(tname, DECAY, G, X, clean, D, 2, dev, None, None)
            assert not np.isfinite(DX.f64()[:row, 1]).any() and not np.isfinite(DH0.f64()[0, 1])
            assert np.isfinite(np.delete(DX.f64(), 1, 1)).all() and np.isfinite(DX.f64()[row:, 1]).all()
            assert np.isfinite(DH0.f64()[1]).all()


@gpu
def test_extreme_gates():
    # large gates on a state of zero: the overflowing product of the gates does not reach it
    for rows in (300, 20000):
        G, X = Mat(np.full((rows, 40), 4.0), torch.float32), Mat(np.zeros((rows, 40)), torch.float32)
        H, L = _scan("f32", DECAY, G, X, 1, None, None)
        assert not H.f64().any() and not L.f64().any()
    # saturated and infinite sigmoid arguments: f is 1 or 0 exactly, nothing is NaN
    g = np.array([[90.0, -90.0, np.inf, -np.inf, 1e30, -1e30, 0.0, 30.0]] * 4)
    for tname in ("f32", "f64", "bf16"):
        G, X = Mat(g, TYPES[tname][0]), Mat(np.ones((4, 8)), TYPES[tname][0])
        H0 = Mat(np.full((1, 8), 2.0), wide(TYPES[tname][0]))
        h = _scan(tname, SIGMOID, G, X, 1, None, H0)[0].f64()
        assert (h[:, [0, 2, 4]] == 2).all() and (h[:, [1, 3, 5]] == 1).all() and np.isfinite(h).all()


@gpu
@pytest.mark.parametrize("rows,cols", [(500, 66), (20000, 5), (300, 33)])
def test_result_in_the_place_of_an_operand(rows, cols):
    for tname in ("f32", "bf16"):
        off, _ = _offsets(rows, 1)
        G, X, H0 = _inputs(tname, SIGMOID, rows, cols, off)
        H, _ = _scan(tname, SIGMOID, G, X, 1, None, H0)
        exp = H.view.clone()
        g0 = G.buf.clone()
        _scan(tname, SIGMOID, G, X, 1, None, H0, H=G)
        assert torch.equal(G.view, exp)
        G.buf.copy_(g0)
        _scan(tname, SIGMOID, G, X, 1, None, H0, H=X, last=False)
        assert torch.equal(X.view, exp)


@gpu
@pytest.mark.parametrize("rows,cols,off", [(130, 70, [0, 0, 50, 130]), (20000, 5, 1), (9001, 34, [0, 1500, 1501, 9000])])
def test_last_states_in_the_place_of_the_first(rows, cols, off):
    off, dev = _offsets(rows, off)
    seqs = len(off) - 1
    for tname in ALL:
        t, code = TYPES[tname]
        G, X, H0 = _inputs(tname, SIGMOID, rows, cols, off)
        H, L = _scan(tname, SIGMOID, G, X, seqs, dev, H0)
        exp, last = H.view.clone(), L.view.clone()
        n = lib.db2k_gated_scan_scratch_bytes(code, rows, cols, seqs)
        s = scratch(n)
        check(lib.db2k_gated_scan(code, SIGMOID, *G.at, *X.at, rows, cols, None if dev is None else dev.data_ptr(), seqs,
                                  *H0.at, *H.at, *H0.at, s.data_ptr(), n, stream()))
        assert torch.equal(H.view, exp) and torch.equal(H0.view, last) and H0.guards_intact()


@gpu
def test_offsets_that_break_their_rules_stay_within_the_matrices():
    G, X, H0 = _inputs("f32", DECAY, 100, 40, np.arange(5))
    dev = torch.tensor([-50, 40, 20, 1 << 40, 90], dtype=torch.int64, device="cuda")
    H, L = _scan("f32", DECAY, G, X, 4, dev, H0)
    torch.cuda.synchronize()
    assert H.guards_intact() and L.guards_intact()


@gpu
@pytest.mark.parametrize("rows,cols,off", [(700, 96, [0, 64, 130, 131, 500, 650]), (20000, 5, 1)])
def test_captured_calls(rows, cols, off):
    off, dev = _offsets(rows, off)
    seqs = len(off) - 1
    t, code = TYPES["bf16"]
    G, X, H0 = _inputs("bf16", SIGMOID, rows, cols, off)
    D = Mat(np.random.default_rng(1).standard_normal((rows, cols)), t)
    H, L = Mat.empty(rows, cols, t), Mat.empty(seqs, cols, wide(t))
    DG, DX, DH0 = Mat.empty(rows, cols, t), Mat.empty(rows, cols, t), Mat.empty(seqs, cols, wide(t))
    n = lib.db2k_gated_scan_scratch_bytes(code, rows, cols, seqs)
    s = scratch(n)
    o = None if dev is None else dev.data_ptr()

    def both():
        check(lib.db2k_gated_scan(code, SIGMOID, *G.at, *X.at, rows, cols, o, seqs, *H0.at, *H.at, *L.at, s.data_ptr(), n,
                                  stream()))
        check(lib.db2k_gated_scan_grad(code, SIGMOID, *G.at, *X.at, *H.at, *D.at, rows, cols, o, seqs, *H0.at, *L.at,
                                       *DG.at, *DX.at, *DH0.at, s.data_ptr(), n, stream()))
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    X.view.normal_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    got = [m.view.clone() for m in (H, L, DG, DX, DH0)]
    both()
    assert all(torch.equal(a, m.view) for a, m in zip(got, (H, L, DG, DX, DH0)))


@gpu
def test_on_handles(ctx):
    import daphne_b200.kernels as k
    rng = np.random.default_rng(3)
    g, x, d = (rng.standard_normal((50, 9)) for _ in range(3))
    h0, dl = rng.standard_normal((3, 9)), rng.standard_normal((3, 9))
    off = np.array([[2], [20], [20], [45]])
    M = lambda a: k.DenseMatrix.from_numpy(ctx, a)  # noqa: E731
    G, X, D, H0, DL, OFF = M(g), M(x), M(d), M(h0), M(dl), M(off)
    h, last = k.gatedScan(k.Gate.SIGMOID, G, X, OFF, H0)
    exp = np.zeros((50, 9))
    for s in range(3):
        v = h0[s]
        for r in range(off[s, 0], off[s + 1, 0]):
            f = 1 / (1 + np.exp(-g[r]))
            v = f * v + (1 - f) * x[r]
            exp[r] = v
        np.testing.assert_allclose(last.to_numpy()[s], v, rtol=0, atol=1e-14)
    np.testing.assert_allclose(h.to_numpy(), exp, rtol=0, atol=1e-14)
    dg, dx, dh0 = k.gatedScanGrad(k.Gate.SIGMOID, G, X, h, D, OFF, H0, DL)
    assert not dg.to_numpy()[[0, 1, 45, 49]].any() and dh0.shape == (3, 9)
    np.testing.assert_allclose(dh0.to_numpy()[1], dl[1], rtol=0, atol=0)  # the empty sequence
    # cumulative sums are the recurrence with gates of one
    ones = k.fill(ctx, 1.0, 50, 9)
    np.testing.assert_allclose(k.gatedScan(k.Gate.DECAY, ones, X)[0].to_numpy(),
                               k.aggCum(k.AggOpCode.SUM, X).to_numpy(), rtol=0, atol=1e-13)
    # steps bring a state up to date in place; another handle of its old values keeps them
    S = k.castObj(H0, np.float64)
    old = k.ewBinaryObjSca(k.BinaryOpCode.ADD, S, 0.0)
    y = k.gatedStep(k.Gate.DECAY, k.sliceRow(G, 0, 3), k.sliceRow(X, 0, 3), S)
    np.testing.assert_allclose(S.to_numpy(), g[:3] * h0 + x[:3], rtol=0, atol=1e-15)
    assert np.array_equal(y.to_numpy(), S.to_numpy()) and np.array_equal(old.to_numpy(), h0)
    G16, X16 = k.castObj(G, np.float16), k.castObj(X, np.float16)
    h16, l16 = k.gatedScan(k.Gate.SIGMOID, G16, X16, OFF, k.castObj(H0, np.float32))
    assert h16.dtype == np.float16 and l16.dtype == np.float32
    np.testing.assert_allclose(h16.to_numpy().astype(np.float64), exp, rtol=0, atol=0.02)
    bad = off.copy()
    for values in ([2, 20, 19, 45], [2, 20, 20, 51], [-1, 20, 20, 45]):
        bad[:, 0] = values
        with pytest.raises(Db2Error, match="offsets must ascend"):
            k.gatedScan(k.Gate.SIGMOID, G, X, M(bad), H0)
    for call, msg in ((lambda: k.gatedScan(7, G, X), "unknown gate"),
                      (lambda: k.gatedScan(k.Gate.DECAY, G, k.sliceRow(X, 0, 5)), "x must have the shape"),
                      (lambda: k.gatedScan(k.Gate.DECAY, G, X, OFF, k.sliceRow(H0, 0, 2)), "h0 must have one row"),
                      (lambda: k.gatedScan(k.Gate.DECAY, G16, X16, None, k.sliceRow(H0, 0, 1)), "wide value type"),
                      (lambda: k.gatedScan(k.Gate.DECAY, G, X, H0), "offsets must be a column"),
                      (lambda: k.gatedScanGrad(k.Gate.DECAY, G, X, h, k.sliceRow(D, 0, 5)), "grad must have"),
                      (lambda: k.gatedScanGrad(k.Gate.SIGMOID, G, None, h, D), "null argument"),
                      (lambda: k.gatedStep(k.Gate.DECAY, G, X, H0), "state must have one row")):
        with pytest.raises(Db2Error, match=msg):
            call()


def test_refusals():
    buf = (C.c_char * 8192)()
    p = C.addressof(buf)
    p += -p % 16

    def refused(code, call):
        with pytest.raises(Db2Error) as e:
            check(call())
        assert e.value.code == code, e.value
    base = dict(dt=names.BF16, gate=SIGMOID, g=p, gld=8, x=p, xld=8, rows=4, cols=8, off=None, seqs=2, h0=p, h0ld=8, h=p,
                hld=8, last=p, lld=8, s=p, sb=8192, d=p, dld=8, dl=p, dlld=8, dg=p, dgld=8, dx=p, dxld=8, dh0=p, dh0ld=8)

    def scan(**kw):
        a = {**base, **kw}
        return lib.db2k_gated_scan(a["dt"], a["gate"], a["g"], a["gld"], a["x"], a["xld"], a["rows"], a["cols"], a["off"],
                                   a["seqs"], a["h0"], a["h0ld"], a["h"], a["hld"], a["last"], a["lld"], a["s"], a["sb"], None)

    def grad(**kw):
        a = {**base, **kw}
        return lib.db2k_gated_scan_grad(a["dt"], a["gate"], a["g"], a["gld"], a["x"], a["xld"], a["h"], a["hld"], a["d"],
                                        a["dld"], a["rows"], a["cols"], a["off"], a["seqs"], a["h0"], a["h0ld"], a["dl"],
                                        a["dlld"], a["dg"], a["dgld"], a["dx"], a["dxld"], a["dh0"], a["dh0ld"], a["s"],
                                        a["sb"], None)

    def step(**kw):
        a = {**base, **kw}
        return lib.db2k_gated_step(a["dt"], a["gate"], a["g"], a["gld"], a["x"], a["xld"], a["rows"], a["cols"], a["h0"],
                                   a["h0ld"], a["last"], a["lld"], a["h"], a["hld"], None)
    for f in (scan, grad, step):
        for dt in (names.I64, names.F8E4M3, 77):
            refused(4, lambda: f(dt=dt))
        for kw in (dict(gate=2), dict(gate=-1), dict(rows=-1), dict(cols=-1), dict(g=None), dict(x=None), dict(gld=7),
                   dict(xld=7), dict(hld=7), dict(h0ld=7)):
            refused(1, lambda: f(**kw))
        assert f(cols=0) == 0
    for f in (scan, grad):
        refused(1, lambda: f(seqs=3))  # 4 rows are not 3 equal sequences
        refused(1, lambda: f(seqs=-1))
        refused(1, lambda: f(h=None))
        long = dict(rows=1 << 20, seqs=1, cols=8)  # cut into blocks: scratch is needed
        assert lib.db2k_gated_scan_scratch_bytes(names.BF16, 1 << 20, 8, 1) > 8192
        for kw in (dict(s=None), dict(s=p + 8, sb=1 << 30), dict(sb=8)):
            refused(1, lambda: f(**long, **kw))
        assert f(seqs=0, rows=0) == 0
    for kw in (dict(d=None), dict(dg=None), dict(dx=None), dict(dld=7), dict(dgld=7), dict(dxld=7), dict(dlld=7),
               dict(dh0ld=7)):
        refused(1, lambda: grad(**kw))
    refused(1, lambda: scan(lld=7))
    refused(1, lambda: step(last=None))
    assert lib.db2k_gated_scan_scratch_bytes(names.F32, 100, 0, 1) == 0
