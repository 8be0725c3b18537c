"""Sums of whole numbers that 32 bits hold exactly: whatever the order of the additions, every result is the exact sum, rounded
once to the value type, so that a part that is lost, taken twice or taken from elsewhere shows."""
import numpy as np
import pytest
import torch

from daphne_b200 import lib as names
from daphne_b200.lib import check, lib
from tests.seq_util import ALL, TYPES, Mat, scratch, stream, wide

pytestmark = pytest.mark.gpu


def _rounded(exact, t):
    """Whole numbers below 2^24 are floats; one rounding to nearest even from there."""
    assert np.abs(exact).max(initial=0) < 2 ** 24
    return torch.as_tensor(exact).float().to(t) if t != torch.float64 else torch.as_tensor(exact)


def _same(got, exact, t, what):
    exp = _rounded(exact, t)
    assert torch.equal(got.cpu().double(), exp.double()), what


@pytest.mark.parametrize("tname,res_t", [("f64", "f64"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"),
                                         ("f16", "f32")])
@pytest.mark.parametrize("vocab,cols,n,kind", [
    (3, 4, 40000, "one"), (5, 260, 3000, "one"), (1, 1, 513, "one"), (3, 8, 300001, "one"), (50000, 4, 1000003, "skewed"),
    (400, 9, 50000, "skewed"), (70000, 24, 16385, "outside"), (90, 130, 2049, "skewed"), (2, 516, 40961, "two"),
    (1000, 33, 700, "skewed"), (64, 1030, 5000, "two"), (7, 2048, 1000, "skewed"),
])
def test_table_gradient(tname, res_t, vocab, cols, n, kind):
    t, code = TYPES[tname]
    rt, rcode = TYPES[res_t]
    rng = np.random.default_rng(vocab + cols + n)
    tok = {"one": lambda: np.full(n, vocab // 2), "two": lambda: np.where(rng.random(n) < 0.4, 0, vocab - 1),
           "outside": lambda: rng.integers(-1, vocab + 2, n),
           "skewed": lambda: np.minimum((vocab ** rng.random(n)).astype(np.int64), vocab) - 1}[kind]()
    most = 2 if res_t == "f16" else 8  # sums of f16 stay below 65504
    grad = rng.integers(-most, most + 1, (n, cols)).astype(np.float64)
    G, d_tok = Mat(grad, t), torch.as_tensor(tok).cuda()
    exact = np.zeros((vocab, cols))
    ok = (tok >= 0) & (tok < vocab)
    np.add.at(exact, tok[ok], grad[ok])
    nb = lib.db2k_embed_grad_scratch_bytes(code, vocab, cols, n)
    s = scratch(nb)
    for start in (None, rng.integers(-9, 10, (vocab, cols)).astype(np.float64)):
        R = Mat.empty(vocab, cols, rt) if start is None else Mat(start, rt)
        check(lib.db2k_embed_grad(code, *G.at, n, cols, names.I64, d_tok.data_ptr(), 1, 1.0, rcode, R.ptr, vocab, R.ld,
                                  int(start is not None), s.data_ptr(), nb, None, stream()))
        _same(R.view, exact if start is None else exact + start, rt, "overwritten" if start is None else "added")
        assert R.guards_intact()


@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("rows,cols", [(1, 1), (40003, 8), (100000, 24), (5000, 130), (6001, 24), (3001, 1024), (600, 4100),
                                       (150, 12288), (700, 16500), (151, 33000), (9, 40000), (2000, 333)])
def test_weight_gradient(tname, rows, cols):
    """dweight is the column sums of grad * s * rstd: rstd is the caller's, a power of two here."""
    t, code = TYPES[tname]
    rng = np.random.default_rng(rows + cols)
    g, s = (rng.integers(-3, 4, (rows, cols)).astype(np.float64) for _ in range(2))
    r = 2.0 ** rng.integers(-1, 2, (rows, 1))
    G, S, V = Mat(g, t), Mat(s, t), Mat(r, wide(t))
    O, DW = Mat.empty(rows, cols, t), Mat.empty(1, cols, wide(t))
    nb = lib.db2k_rms_norm_grad_scratch_bytes(code, rows, cols)
    check(lib.db2k_rms_norm_grad(code, *G.at, rows, cols, *S.at, None, V.ptr, None, 0, *O.at, DW.ptr, scratch(nb).data_ptr(),
                                 nb, stream()))
    exact = 2 * (g * s * r).sum(0, keepdims=True)
    assert np.abs(exact).max() < 2 ** 24
    assert np.array_equal(2 * DW.f64(), exact)
    assert O.guards_intact() and DW.guards_intact()


@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("rows,cols,off", [
    (1, 1, 1), (64, 65, 1), (1000, 70, 1), (2400, 33, 8), (700, 96, [0, 1, 1, 64, 130, 131, 500, 500, 650]), (20000, 5, 1),
    (9001, 34, [0, 1500, 1501, 9000]), (60000, 2, 2), (8192, 1024, 1), (300, 4100, 3), (100000, 96, 1), (5000, 260, [3, 4999]),
])
def test_recurrence_and_its_gradient(tname, rows, cols, off):
    """Gates of 0, 1 and -1 and whole inputs: states are whole, and every sum has one exact value."""
    t, code = TYPES[tname]
    rng = np.random.default_rng(rows + cols)
    off, dev = (np.arange(off + 1) * (rows // off), None) if isinstance(off, int) else (np.array(off), torch.tensor(off).cuda())
    seqs, o = len(off) - 1, None if dev is None else dev.data_ptr()
    g = rng.choice([1.0, -1.0, 0.0], (rows, cols), p=[0.94, 0.05, 0.01])
    x, d = (rng.integers(-4, 5, (rows, cols)).astype(np.float64) for _ in range(2))
    h0, dl = (rng.integers(-9, 10, (seqs, cols)).astype(np.float64) for _ in range(2))
    G, X, D, H0, DL = Mat(g, t), Mat(x, t), Mat(d, t), Mat(h0, wide(t)), Mat(dl, wide(t))
    H, DG, DX = (Mat.empty(rows, cols, t) for _ in range(3))
    L, DH0 = Mat.empty(seqs, cols, wide(t)), Mat.empty(seqs, cols, wide(t))
    nb = lib.db2k_gated_scan_scratch_bytes(code, rows, cols, seqs)
    s = scratch(nb)
    check(lib.db2k_gated_scan(code, names.GATE_DECAY, *G.at, *X.at, rows, cols, o, seqs, *H0.at, *H.at, *L.at, s.data_ptr(), nb,
                              stream()))
    h, last, delta, dh0 = np.zeros((rows, cols)), np.zeros((seqs, cols)), np.zeros((rows, cols)), np.zeros((seqs, cols))
    inside = np.zeros(rows, dtype=bool)
    for q in range(seqs):
        v, c = h0[q], dl[q]
        for r in range(off[q], off[q + 1]):
            v = g[r] * v + x[r]
            h[r], inside[r] = v, True
        last[q] = v
        for r in range(off[q + 1] - 1, off[q] - 1, -1):
            delta[r] = d[r] + c
            c = g[r] * delta[r]
        dh0[q] = c
    _same(H.view[torch.as_tensor(inside).cuda()], h[inside], t, "h")
    _same(L.view, last, wide(t), "last")
    # any whole h: the gradient reads the one that it is given
    some = rng.integers(-4, 5, (rows, cols)).astype(np.float64)
    HG = Mat(some, t)
    check(lib.db2k_gated_scan_grad(code, names.GATE_DECAY, *G.at, None, 0, *HG.at, *D.at, rows, cols, o, seqs, *H0.at, *DL.at,
                                   *DG.at, *DX.at, *DH0.at, s.data_ptr(), nb, stream()))
    above = np.vstack([np.zeros((1, cols)), some[:-1]])
    for q in range(seqs):
        if off[q] < off[q + 1]:
            above[off[q]] = h0[q]
    _same(DX.view[torch.as_tensor(inside).cuda()], delta[inside], t, "dx")
    _same(DG.view[torch.as_tensor(inside).cuda()], (delta * above)[inside], t, "dg")
    _same(DH0.view, dh0, wide(t), "dh0")
    assert all(m.guards_intact() for m in (H, L, DG, DX, DH0))
