"""Embedding lookup and its gradient by sorted tokens against plain 64-bit loops.

Tolerances: a lookup is one product in the wide type (the scale rounded once, the product once) and one rounding to the
type.  A sum of m terms in any order is off by at most (m - 1) steps of the sum of the magnitudes (first order), one
more rounding each for the scale and the product, one for the type."""
import ctypes as C

import numpy as np
import pytest
import torch

from daphne_b200 import lib as names
from daphne_b200.lib import Db2Error, check, lib
from tests.seq_util import ALL, GUARD, TYPES, Mat, assert_within, half_step, scratch, smallest, stream, wide

gpu = pytest.mark.gpu
INDEX = {"i64": (torch.int64, names.I64), "i32": (torch.int32, names.I32)}


def _tokens(rng, n, vocab, kind):
    if kind == "uniform":
        t = rng.integers(0, vocab, n)
    elif kind == "one":
        t = np.full(n, vocab // 2)
    elif kind == "skewed":
        t = np.minimum((vocab ** rng.random(n)).astype(np.int64), vocab) - 1
    else:  # padding and values outside the table
        t = rng.integers(-1, vocab + 2, n)
    return t.astype(np.int64)


def _lookup(tname, table, tok, scale, index="i64", tok_ld=1, pad=0, shift=0, status=None):
    t, code = TYPES[tname]
    T = Mat(table, t, pad, shift)
    it, icode = INDEX[index]
    d_tok = torch.zeros(max(len(tok), 1) * tok_ld, dtype=it, device="cuda")
    d_tok[::tok_ld][:len(tok)] = torch.as_tensor(tok).to(it).cuda()
    R = Mat.empty(len(tok), T.cols, t, pad, shift)
    check(lib.db2k_embed(code, T.ptr, T.rows, T.cols, T.ld, icode, d_tok.data_ptr(), tok_ld, len(tok), scale, R.ptr, R.ld,
                         None if status is None else status.data_ptr(), stream()))
    return T, R


@gpu
@pytest.mark.parametrize("tname", ALL)
@pytest.mark.parametrize("vocab,cols,n,pad,shift,index,tok_ld,kind", [
    (1, 1, 1, 0, 0, "i64", 1, "uniform"),
    (5, 7, 3, 0, 0, "i32", 1, "uniform"),
    (100, 64, 1000, 0, 0, "i64", 1, "outside"),
    (333, 129, 257, 7, 0, "i32", 3, "outside"),      # rows end inside a packet, aligned rows for the 16-bit types
    (50, 515, 70, 0, 1, "i64", 2, "skewed"),         # nothing aligned
    (64, 4100, 9, 4, 8, "i64", 1, "uniform"),        # few rows, cut along the columns
    (9, 20000, 2, 0, 0, "i64", 1, "uniform"),
    (17, 24, 40001, 8, 16, "i32", 1, "skewed"),
    (77, 130, 300, 0, 0, "i64", 1, "outside"),       # pairs
    (20, 1030, 40, 2, 2, "i64", 1, "uniform"),
])
def test_lookup(tname, vocab, cols, n, pad, shift, index, tok_ld, kind):
    rng = np.random.default_rng(vocab + cols + n)
    tok = _tokens(rng, n, vocab, kind)
    scale = 1.7
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    T, R = _lookup(tname, rng.standard_normal((vocab, cols)), tok, scale, index, tok_ld, pad, shift, status)
    t = TYPES[tname][0]
    ok = (tok >= 0) & (tok < vocab)
    exp = np.where(ok[:, None], T.f64()[np.where(ok, tok, 0)] * scale, 0.0)
    assert_within(R.f64(), exp, np.abs(exp) * (half_step(t) + 3 * half_step(wide(t))) + smallest(t), "embed")
    assert R.guards_intact() and T.guards_intact()
    assert int(status) == int((~ok & (tok != -1)).any())


@gpu
def test_lookup_scale_one_copies_bits_and_non_finite_values():
    table = np.array([[np.inf, -np.inf, np.nan, -0.0, 1.5, 6e-8, 60000.0, -2.0]])
    for tname in ALL:
        T, R = _lookup(tname, table, np.array([0, 0]), 1.0)
        t = TYPES[tname][0]
        size = {8: torch.int64, 4: torch.int32, 2: torch.int16}[t.itemsize]
        for r in range(2):
            got, exp = R.view[r], T.view[0]
            same = got.view(size) == exp.view(size)
            assert bool((same | (got.isnan() & exp.isnan())).all()), tname


def _grad(tname, grad, tok, vocab, scale, res=None, res_t=None, index="i64", pad=0, shift=0, status=None, accumulate=0):
    t, code = TYPES[tname]
    rt, rcode = TYPES[res_t or tname]
    G = Mat(grad, t, pad, shift)
    it, icode = INDEX[index]
    d_tok = torch.as_tensor(tok).to(it).cuda()
    R = res if res is not None else Mat.empty(vocab, G.cols, rt, pad, shift)
    n = lib.db2k_embed_grad_scratch_bytes(code, vocab, G.cols, len(tok))
    s = scratch(n)
    check(lib.db2k_embed_grad(code, G.ptr, G.ld, len(tok), G.cols, icode, d_tok.data_ptr(), 1, scale, rcode, R.ptr, vocab,
                              R.ld, accumulate, s.data_ptr(), n, None if status is None else status.data_ptr(), stream()))
    return G, R


def _expect(G, tok, vocab, scale):
    g, ok = G.f64(), (tok >= 0) & (tok < vocab)
    exp, mag = np.zeros((vocab, G.cols)), np.zeros((vocab, G.cols))
    np.add.at(exp, tok[ok], g[ok])
    np.add.at(mag, tok[ok], np.abs(g[ok]))
    m = np.bincount(tok[ok], minlength=vocab)[:, None]
    return exp * scale, mag * scale, m


@gpu
@pytest.mark.parametrize("tname,res_t", [("f64", "f64"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"),
                                         ("f16", "f32")])
@pytest.mark.parametrize("vocab,cols,n,pad,shift,index,kind", [
    (1, 1, 1, 0, 0, "i64", "uniform"),
    (7, 3, 33, 0, 0, "i32", "uniform"),
    (1000, 40, 65, 0, 0, "i64", "uniform"),          # most rows untouched
    (33, 64, 3000, 8, 8, "i64", "outside"),
    (500, 130, 4097, 3, 1, "i64", "skewed"),
    (5, 2000, 1000, 0, 0, "i32", "one"),             # one token: every run holds a part of one sum
    (90, 16, 1024, 0, 0, "i64", "skewed"),           # one chunk of the sort, and one token more
    (90, 16, 1025, 0, 0, "i32", "outside"),
    (3000, 12, 9001, 0, 0, "i64", "skewed"),         # nine chunks
    (70000, 16, 16384, 0, 0, "i64", "skewed"),       # sixteen chunks, no remainder
    (70000, 24, 16385, 0, 0, "i64", "outside"),
    (70000, 8, 40960, 0, 0, "i64", "skewed"),        # the most tokens that are merged, and one more for the radix passes
    (70000, 8, 40961, 0, 0, "i64", "outside"),
    (300000, 8, 45001, 0, 0, "i64", "skewed"),       # three passes
    (400, 9, 50000, 1, 0, "i32", "skewed"),          # one pass
    (3, 4, 40000, 0, 0, "i64", "one"),
    (50, 130, 2000, 0, 0, "i64", "skewed"),          # pairs
    (50, 258, 900, 2, 2, "i64", "outside"),
    (1000, 33, 700, 0, 1, "i64", "skewed"),          # a contiguous table off 16-byte boundaries
    (1000, 33, 700, 0, 0, "i64", "skewed"),          # and on one, with bytes behind the last whole packet
    (3, 4, 30000, 0, 0, "i64", "one"),
])
def test_gradient(tname, res_t, vocab, cols, n, pad, shift, index, kind):
    rng = np.random.default_rng(vocab + cols + n)
    tok = _tokens(rng, n, vocab, kind)
    scale = 0.6
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    grad = rng.standard_normal((n, cols))
    G, R = _grad(tname, grad, tok, vocab, scale, None, res_t, index, pad, shift, status)
    t, rt = TYPES[tname][0], TYPES[res_t][0]
    exp, mag, m = _expect(G, tok, vocab, scale)
    bound = np.abs(exp) * half_step(rt) + mag * (m + 3) * half_step(wide(t)) + smallest(rt)
    assert_within(R.f64(), exp, bound, "embedGrad")
    assert R.guards_intact() and G.guards_intact()
    assert int(status) == int(((tok < -1) | (tok >= vocab)).any())
    # the same bits again, and the sums added to what is there
    _, again = _grad(tname, grad, tok, vocab, scale, None, res_t, index, pad, shift)
    assert torch.equal(again.view, R.view)
    start = rng.standard_normal((vocab, cols))
    A = Mat(start, rt, pad, shift)
    before = A.f64()
    _grad(tname, grad, tok, vocab, scale, A, res_t, index, pad, shift, accumulate=1)
    exp2 = before + exp
    assert_within(A.f64(), exp2, np.abs(exp2) * half_step(rt) + (mag * (m + 3) + np.abs(before) + mag) * half_step(wide(t)) +
                  smallest(rt), "added")
    assert A.guards_intact()
    untouched = m[:, 0] == 0
    assert np.array_equal(A.f64()[untouched], before[untouched])


@gpu
def test_gradient_of_many_tokens_and_of_none():
    rng = np.random.default_rng(3)
    tok = _tokens(rng, 1_000_003, 50000, "skewed")
    G, R = _grad("f32", rng.standard_normal((len(tok), 4)), tok, 50000, 1.0)
    exp, mag, m = _expect(G, tok, 50000, 1.0)
    # runs of 32 terms, their sums added in eight shares: far fewer roundings in a row than terms, m is a safe bound
    assert_within(R.f64(), exp, np.abs(exp) * 2.0 ** -24 + mag * (m + 3) * 2.0 ** -24, "embedGrad 1M")
    _, Z = _grad("f32", np.zeros((0, 4)), np.zeros(0, dtype=np.int64), 100, 1.0, pad=2)
    assert not Z.f64().any()
    keep = Mat(rng.standard_normal((100, 4)), torch.float32)
    before = keep.f64()
    _grad("f32", np.zeros((0, 4)), np.zeros(0, dtype=np.int64), 100, 1.0, res=keep, accumulate=1)
    assert np.array_equal(keep.f64(), before)


@gpu
def test_gradient_agrees_with_differences():
    """d/dE of f(E) = sum(w * embed(E)) against central differences (f is linear: exact up to rounding)."""
    rng = np.random.default_rng(4)
    vocab, cols, n = 6, 5, 40
    tok = rng.integers(0, vocab, n)
    E, w = rng.standard_normal((vocab, cols)), rng.standard_normal((n, cols))

    def f(table):
        return float((_lookup("f64", table, tok, 1.3)[1].f64() * w).sum())

    _, R = _grad("f64", w, tok, vocab, 1.3)
    got, step = R.f64(), 1e-3
    for v in range(vocab):
        for c in range(cols):
            d = np.zeros_like(E)
            d[v, c] = step
            diff = (f(E + d) - f(E - d)) / (2 * step)
            # each f is a sum of 200 terms of about one: 200 * 200 * 2^-53 off, divided by 2 * step
            assert abs(diff - got[v, c]) < 200 * 200 * 2.0 ** -52 / step


@gpu
def test_captured_calls_replay_with_new_inputs_beside_other_streams():
    rng = np.random.default_rng(5)
    vocab, cols, n = 500, 96, 3000
    t, code = TYPES["bf16"]
    table = Mat(rng.standard_normal((vocab, cols)), t)
    tok = torch.as_tensor(_tokens(rng, n, vocab, "skewed")).cuda()
    y, grad, d = Mat.empty(n, cols, t), Mat(rng.standard_normal((n, cols)), t), Mat.empty(vocab, cols, torch.float32)
    nb = lib.db2k_embed_grad_scratch_bytes(code, vocab, cols, n)
    s = scratch(nb)

    def both():
        check(lib.db2k_embed(code, *table.at[:1], vocab, cols, cols, names.I64, tok.data_ptr(), 1, n, 2.0, *y.at, None,
                             stream()))
        check(lib.db2k_embed_grad(code, *grad.at, n, cols, names.I64, tok.data_ptr(), 1, 2.0, names.F32, d.ptr, vocab,
                                  d.ld, 0, s.data_ptr(), nb, None, stream()))

    both()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        both()
    for k in range(2):
        tok.copy_(torch.as_tensor(_tokens(rng, n, vocab, "uniform" if k else "outside")).cuda())
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            g.replay()
        side.synchronize()
        gy, gd = y.view.clone(), d.view.clone()
        both()
        torch.cuda.synchronize()
        assert torch.equal(gy, y.view) and torch.equal(gd, d.view)


@gpu
def test_on_handles(ctx):
    import daphne_b200.kernels as k
    rng = np.random.default_rng(6)
    E, tok = rng.standard_normal((40, 12)), rng.integers(-1, 40, (100, 1))
    dE, dt = k.DenseMatrix.from_numpy(ctx, E), k.DenseMatrix.from_numpy(ctx, tok)
    got = k.embed(dE, dt, 3.0).to_numpy()
    exp = np.where(tok >= 0, E[np.maximum(tok[:, 0], 0)] * 3.0, 0.0)
    assert np.array_equal(got, exp)
    # rows and columns of a view, a deferred chain as the table, the product with one-hot rows
    view = k.sliceCol(k.sliceRow(dE, 5, 30), 3, 10)
    few = np.minimum(tok, 24)
    assert np.array_equal(k.embed(view, k.DenseMatrix.from_numpy(ctx, few)).to_numpy(),
                          np.where(few >= 0, E[5:30, 3:10][np.maximum(few[:, 0], 0)], 0.0))
    twice = k.ewBinaryObjSca(k.BinaryOpCode.MUL, dE, 2.0)
    assert np.array_equal(k.embed(twice, dt).to_numpy(), np.where(tok >= 0, 2.0 * E[np.maximum(tok[:, 0], 0)], 0.0))
    G = rng.standard_normal((100, 12))
    dG = k.DenseMatrix.from_numpy(ctx, G)
    ref = np.zeros((40, 12))
    np.add.at(ref, tok[tok[:, 0] >= 0, 0], G[tok[:, 0] >= 0])
    grad = k.embedGrad(dG, dt, 40)
    np.testing.assert_allclose(grad.to_numpy(), ref, rtol=0, atol=100 * 100 * 2.0 ** -53)
    grad2 = k.embedGrad(dG, dt, 40, add_to=grad)
    assert grad2 is grad
    np.testing.assert_allclose(grad.to_numpy(), 2 * ref, rtol=0, atol=300 * 100 * 2.0 ** -53)
    # adding to a matrix whose buffer a second handle reads leaves that handle's values alone
    u = k.DenseMatrix.from_numpy(ctx, np.arange(480, dtype=np.float64).reshape(40, 12))
    chain = k.ewBinaryObjSca(k.BinaryOpCode.ADD, u, 1.0)
    k.embedGrad(dG, dt, 40, add_to=u)
    assert np.array_equal(chain.to_numpy(), np.arange(480).reshape(40, 12) + 1.0)
    # 16-bit matrices and a float gradient of them
    hE = k.castObj(dE, k.BFLOAT16)
    hy = k.castObj(k.embed(hE, dt), np.float64).to_numpy()
    bits = torch.as_tensor(E).to(torch.bfloat16).double().numpy()
    assert np.array_equal(hy, np.where(tok >= 0, bits[np.maximum(tok[:, 0], 0)], 0.0))
    f = k.embedGrad(k.castObj(dG, np.float16), dt, 40, dtype=np.float32)
    assert f.dtype == np.float32
    np.testing.assert_allclose(f.to_numpy(), ref, rtol=0, atol=100 * 4 * 2.0 ** -10)
    for bad in (40, -2):
        t2 = tok.copy()
        t2[50, 0] = bad
        with pytest.raises(Db2Error, match="outside the 40 rows"):
            k.embed(dE, k.DenseMatrix.from_numpy(ctx, t2))
        with pytest.raises(Db2Error, match="outside the 40 rows"):
            k.embedGrad(dG, k.DenseMatrix.from_numpy(ctx, t2), 40)
    assert np.array_equal(k.embed(dE, dt, 3.0).to_numpy(), exp)  # the context goes on
    with pytest.raises(Db2Error, match="column matrix"):
        k.embed(dE, dG)
    with pytest.raises(Db2Error, match="as many rows"):
        k.embedGrad(dG, k.DenseMatrix.from_numpy(ctx, tok[:50]), 40)
    with pytest.raises(Db2Error, match="expected"):
        k.embedGrad(dG, dt, 41, add_to=u)
    with pytest.raises(Db2Error, match="int64 or int32"):
        k.embed(dE, k.DenseMatrix.from_numpy(ctx, E[:, :1].copy()))


def test_refusals():
    """Argument checks come before anything touches a device."""
    buf = (C.c_char * 4096)()
    p = C.addressof(buf)
    p += -p % 16

    def refused(code, call):
        with pytest.raises(Db2Error) as e:
            check(call())
        assert e.value.code == code, e.value
    F, I = names.BF16, names.I64
    ok = dict(dt=F, table=p, vocab=4, cols=8, ld=8, it=I, tok=p, tld=1, n=3, res=p, rld=8)

    def emb(**kw):
        a = {**ok, **kw}
        return lib.db2k_embed(a["dt"], a["table"], a["vocab"], a["cols"], a["ld"], a["it"], a["tok"], a["tld"], a["n"], 1.0,
                              a["res"], a["rld"], None, None)
    for dt in (names.I64, names.U8, names.F8E4M3, 99):
        refused(4, lambda: emb(dt=dt))
    refused(4, lambda: emb(it=names.U64))
    for kw in (dict(vocab=-1), dict(cols=-1), dict(n=-1), dict(table=None), dict(tok=None), dict(res=None), dict(ld=7),
               dict(rld=7), dict(tld=0)):
        refused(1, lambda: emb(**kw))
    assert emb(n=0, res=None) == 0 and emb(cols=0) == 0
    ok = dict(dt=F, grad=p, gld=8, n=3, cols=8, it=I, tok=p, tld=1, rdt=F, res=p, vocab=4, rld=8, s=p, sb=1 << 20)

    def grad(**kw):
        a = {**ok, **kw}
        return lib.db2k_embed_grad(a["dt"], a["grad"], a["gld"], a["n"], a["cols"], a["it"], a["tok"], a["tld"], 1.0,
                                   a["rdt"], a["res"], a["vocab"], a["rld"], 0, a["s"], a["sb"], None, None)
    for kw in (dict(dt=names.U8), dict(rdt=names.F16), dict(rdt=names.F64), dict(it=names.F32), dict(n=1 << 31),
               dict(vocab=(1 << 31) - 1)):
        refused(4, lambda: grad(**kw))
    for kw in (dict(n=-1), dict(grad=None), dict(tok=None), dict(res=None), dict(gld=7), dict(rld=7), dict(s=None),
               dict(s=p + 8), dict(sb=16)):
        refused(1, lambda: grad(**kw))
    assert grad(vocab=0) == 0 and grad(cols=0) == 0
    assert lib.db2k_embed_grad_scratch_bytes(F, 4, 8, 0) == 0
