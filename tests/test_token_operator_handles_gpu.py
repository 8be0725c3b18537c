"""The handle forms of the operators on sequences of tokens: results that name their operands, calls that are refused, and
what is left behind then."""
import ctypes as C

import numpy as np
import pytest

from daphne_b200.lib import check, lib

gpu = pytest.mark.gpu
SHAPE = (260, 300)  # chains on doubles of at least 65536 elements are deferred


@gpu
@pytest.mark.parametrize("dtype", [np.float64, np.float32])
@pytest.mark.parametrize("kind", ["host only", "on the device", "deferred", "shared"])
@pytest.mark.parametrize("slot", ["new", "given", "in place"])
def test_step_whose_result_names_the_state(ctx, dtype, kind, slot):
    """h over the state, or the new state over it, whatever the state's values lie in; other handles keep the old values."""
    import daphne_b200.kernels as k
    rng = np.random.default_rng(1)
    g, x, s = (rng.integers(-8, 9, SHAPE).astype(dtype) for _ in range(3))
    G, X, S = (k.DenseMatrix.from_numpy(ctx, a) for a in (g, x, s))
    other = None
    if kind == "on the device":
        S.device_ptr()
    elif kind == "deferred":
        S = k.ewBinaryObjSca(k.BinaryOpCode.MUL, S, 2.0)
        s = s * 2
    elif kind == "shared":
        other = k.ewBinaryObjSca(k.BinaryOpCode.ADD, S, 0.0)
    junk = k.fill(ctx, 77.0, *SHAPE, dtype=dtype)  # memory that a fresh buffer may come from
    junk.device_ptr()
    del junk
    exp = g * s + x  # small whole numbers: exact
    if slot == "in place":
        h = C.c_void_p()
        check(lib.db2_gatedStep(ctx.handle, int(k.Gate.DECAY), C.byref(h), C.byref(S._h), G.handle, X.handle, S.handle))
        result, new = k.DenseMatrix(ctx, h), S
    else:
        new = k.fill(ctx, 5.0, *SHAPE, dtype=dtype) if slot == "given" else None
        n = new._h if new is not None else C.c_void_p()
        check(lib.db2_gatedStep(ctx.handle, int(k.Gate.DECAY), C.byref(S._h), C.byref(n), G.handle, X.handle, S.handle))
        result, new = S, new if new is not None else k.DenseMatrix(ctx, n)
    assert np.array_equal(result.to_numpy(), exp) and np.array_equal(new.to_numpy(), exp)
    if other is not None:
        assert np.array_equal(other.to_numpy(), s)


@gpu
def test_tokens_are_checked_where_nothing_is_computed(ctx):
    """No table rows, or no columns: a token that names no row is an error all the same, and -1 is padding."""
    import daphne_b200.kernels as k
    from daphne_b200.lib import Db2Error
    tokens = lambda *t: k.DenseMatrix.from_numpy(ctx, np.array(t, dtype=np.int64).reshape(-1, 1))  # noqa: E731
    for vocab, cols in ((0, 4), (0, 0), (3, 0)):
        for t in (np.float64, np.float16):
            table, grad = k.DenseMatrix.empty(ctx, vocab, cols, t), k.DenseMatrix.empty(ctx, 2, cols, t, zero=True)
            fine = tokens(-1, min(vocab, 3) - 1)
            assert k.embed(table, fine).shape == (2, cols) and k.embedGrad(grad, fine, vocab).shape == (vocab, cols)
            assert k.embed(table, k.castObj(fine, np.int64)).shape == (2, cols)
            for bad in (tokens(-1, vocab), tokens(-2, -1), tokens(5, 7)):
                with pytest.raises(Db2Error, match="outside the %d rows" % vocab):
                    k.embed(table, bad)
                with pytest.raises(Db2Error, match="outside the %d rows" % vocab):
                    k.embedGrad(grad, bad, vocab)
    none = tokens()
    assert k.embed(k.DenseMatrix.empty(ctx, 0, 4), none).shape == (0, 4)
    assert k.embedGrad(k.DenseMatrix.empty(ctx, 0, 4), none, 0).shape == (0, 4)


@gpu
@pytest.mark.parametrize("index", [np.int64, np.int32])
def test_token_status_on_pointers_where_nothing_is_computed(index):
    import torch
    from daphne_b200 import lib as names
    from tests.seq_util import stream
    code = names.I64 if index == np.int64 else names.I32
    tok = torch.as_tensor(np.array([-1, 99, -1, 99, 4, 99], dtype=index)).cuda()  # every second one, and the third is outside
    buf = torch.zeros(64, device="cuda")
    p = buf.data_ptr()
    for n, exp in ((2, 0), (3, 1)):
        for vocab, cols in ((0, 4), (0, 0), (3, 0)):
            st = torch.zeros(2, dtype=torch.int32, device="cuda")
            check(lib.db2k_embed(names.F32, p, vocab, cols, cols, code, tok.data_ptr(), 2, n, 1.0, p if cols == 0 else p + 128,
                                 cols, st.data_ptr(), stream()))
            check(lib.db2k_embed_grad(names.F32, p, cols, n, cols, code, tok.data_ptr(), 2, 1.0, names.F32, p, vocab, cols, 0,
                                      None, 0, st.data_ptr() + 4, stream()))
            assert st.tolist() == [exp, exp], (n, vocab, cols)


def _calls(ctx, k):
    """(The operands, to be kept; every operator with several results: the names of its slots, a call with their values.)"""
    rng = np.random.default_rng(7)
    n, c = 40, 6
    M = lambda r, q=c, t=np.float32: k.DenseMatrix.from_numpy(ctx, rng.standard_normal((r, q)).astype(t))  # noqa: E731
    d, s = int(k.Gate.DECAY), ctx.handle
    off = k.DenseMatrix.from_numpy(ctx, np.array([[0], [15], [40]]))
    x, r, w, v, st, g, last = M(n), M(n), M(1), M(n, 1), M(2), M(n), M(2)
    state = M(n)
    ref = C.byref
    return [x, r, w, v, st, g, last, state, off], {
        "rmsNorm": (["res", "sum", "rstd"], lambda a, b, e: lib.db2_rmsNorm(s, ref(a), ref(b), ref(e), x.handle, r.handle, w.handle, 1e-6)),
        "rmsNormQ8": (["res", "scales", "sum", "rstd"], lambda a, b, e, f: lib.db2_rmsNormQ8(
            s, ref(a), ref(b), ref(e), ref(f), x.handle, r.handle, w.handle, 1e-6, 16)),
        "rmsNormGrad": (["dx", "dweight"], lambda a, b: lib.db2_rmsNormGrad(s, ref(a), ref(b), x.handle, r.handle, w.handle, v.handle, None)),
        "gatedScan": (["h", "last"], lambda a, b: lib.db2_gatedScan(s, d, ref(a), ref(b), g.handle, x.handle, off.handle, st.handle)),
        "gatedScanGrad": (["dg", "dx", "dh0"], lambda a, b, e: lib.db2_gatedScanGrad(
            s, d, ref(a), ref(b), ref(e), g.handle, x.handle, r.handle, x.handle, off.handle, st.handle, last.handle)),
        "gatedStep": (["h", "new_state"], lambda a, b: lib.db2_gatedStep(s, d, ref(a), ref(b), g.handle, x.handle, state.handle)),
    }


@gpu
@pytest.mark.parametrize("name", ["rmsNorm", "rmsNormQ8", "rmsNormGrad", "gatedScan", "gatedScanGrad", "gatedStep"])
def test_a_refused_result_leaves_the_others_as_they_were(ctx, name):
    """Each result in turn has the wrong shape: no other slot is touched, also not one that
    names an operand whose values lie on the host only, and nothing is made."""
    import daphne_b200.kernels as k
    keep, calls = _calls(ctx, k)
    slots, call = calls[name]
    assert call(*[C.c_void_p() for _ in slots]) == 0
    for wrong in range(len(slots)):
        bad = k.fill(ctx, 7.0, 3, 3, dtype=np.float32)
        for over in range(len(slots)):  # which other slot holds a given matrix, whose values have to stay
            given = [C.c_void_p() for _ in slots]
            given[wrong] = C.c_void_p(bad.handle.value)
            own = None
            if over != wrong and slots[over] in ("res", "sum", "dx", "h", "dg", "new_state") and (name, slots[over]) != ("rmsNormQ8", "res"):
                own = k.DenseMatrix.from_numpy(ctx, np.full((40, 6), 3.0, dtype=np.float32))
                given[over] = C.c_void_p(own.handle.value)
            before = [h.value for h in given]
            assert call(*given) == 1, (slots[wrong], over)
            assert [h.value for h in given] == before, (slots[wrong], over)
            assert (bad.to_numpy() == 7).all()
            if own is not None:
                assert (own.to_numpy() == 3).all(), (slots[wrong], slots[over])


@gpu
@pytest.mark.parametrize("name", ["rmsNorm", "rmsNormQ8", "rmsNormGrad", "gatedScan", "gatedScanGrad", "gatedStep"])
def test_one_slot_for_two_results_is_refused(ctx, name):
    import daphne_b200.kernels as k
    keep, calls = _calls(ctx, k)
    slots, call = calls[name]
    for i in range(len(slots)):
        for j in range(i):
            given = [C.c_void_p() for _ in slots]
            given[i] = given[j]
            assert call(*given) == 1 and all(h.value is None for h in given), (slots[i], slots[j])


@gpu
def test_a_token_outside_the_table_leaves_no_result_behind(ctx):
    import daphne_b200.kernels as k
    x = k.DenseMatrix.from_numpy(ctx, np.ones((4, 3)))
    tok = k.DenseMatrix.from_numpy(ctx, np.array([[0], [4], [1], [2]]))
    for call in (lambda h: lib.db2_embed(ctx.handle, C.byref(h), x.handle, tok.handle, 1.0),
                 lambda h: lib.db2_embedGrad(ctx.handle, C.byref(h), x.handle, tok.handle, 4, 1.0, x.dtype_code, 0)):
        h = C.c_void_p()
        assert call(h) == 5 and h.value is None
        given = k.fill(ctx, 2.0, 4, 3)
        h = C.c_void_p(given.handle.value)
        assert call(h) == 5 and h.value == given.handle.value


@gpu
def test_updates_through_a_view_leave_earlier_results_alone(ctx):
    """What was asked for before an update in place has the values of that time, also where it is computed later: chains,
    row aggregations, products of the whole matrix and of other views of it."""
    import daphne_b200.kernels as k
    rng = np.random.default_rng(3)
    p, g, x = (rng.integers(-4, 5, s).astype(np.float64) for s in ((600, 300), (260, 300), (260, 300)))
    tok = rng.integers(0, 260, (50, 1))
    dy = rng.integers(-4, 5, (50, 300)).astype(np.float64)
    M = lambda a: k.DenseMatrix.from_numpy(ctx, a)  # noqa: E731
    for update in ("step", "table gradient"):
        P = M(p)
        P.device_ptr()
        v, other = k.sliceRow(P, 20, 280), k.sliceRow(P, 100, 500)
        twice, less = k.ewBinaryObjSca(k.BinaryOpCode.MUL, P, 2.0), k.ewBinaryMat(k.BinaryOpCode.SUB, other, M(p[100:500]))
        plus = k.ewBinaryMat(k.BinaryOpCode.ADD, M(p * 3), P)
        rows, gram = k.aggRow(k.AggOpCode.SUM, k.ewUnaryMat(k.UnaryOpCode.ABS, P)), k.syrk(P)
        new = p.copy()
        if update == "step":
            k.gatedStep(k.Gate.DECAY, M(g), M(x), v)
            new[20:280] = g * p[20:280] + x
        else:
            k.embedGrad(M(dy), M(tok), 260, add_to=v)
            np.add.at(new, 20 + tok[:, 0], dy)
        assert np.array_equal(P.to_numpy(), new) and np.array_equal(v.to_numpy(), new[20:280])
        assert np.array_equal(twice.to_numpy(), 2 * p) and not less.to_numpy().any() and np.array_equal(plus.to_numpy(), 4 * p)
        assert np.array_equal(rows.to_numpy()[:, 0], np.abs(p).sum(1)) and np.array_equal(gram.to_numpy(), p.T @ p)
        assert np.array_equal(k.ewBinaryObjSca(k.BinaryOpCode.MUL, P, 2.0).to_numpy(), 2 * new)


@gpu
def test_updates_leave_earlier_sparse_products_alone(ctx):
    """A deferred product of a CSR matrix with a dense one has the dense one's values of the time it was asked for."""
    import daphne_b200.kernels as k
    val, col, off = np.ones(6), np.array([0, 2, 1, 0, 1, 2], dtype=np.uint64), np.array([0, 2, 3, 6], dtype=np.uint64)
    full = np.array([[1.0, 0, 1], [0, 1, 0], [1, 1, 1]])
    w, g, x = np.array([[2.0, 3.0, 5.0]]), np.array([[4.0, 4.0, 4.0]]), np.array([[1.0, 1.0, 1.0]])
    M = lambda a: k.DenseMatrix.from_numpy(ctx, a)  # noqa: E731
    for part in (False, True):
        W = M(np.vstack([w, w]) if part else w)
        W.device_ptr()
        v = k.sliceRow(W, 0, 1) if part else W
        G = k.CSRMatrix.from_arrays(ctx, 3, 3, val, col, off)
        prod = k.ewMulCsrDense(G, v)
        k.gatedStep(k.Gate.DECAY, M(g), M(x), v)
        assert np.array_equal(v.to_numpy(), g * w + x)
        assert np.array_equal(k.aggRowCsr(k.AggOpCode.SUM, prod).to_numpy()[:, 0], (full * w).sum(1))


@gpu
def test_updates_leave_a_product_of_a_tall_matrix_with_itself_alone(ctx):
    import daphne_b200.kernels as k
    p = np.random.default_rng(5).integers(-3, 4, (1 << 16, 64)).astype(np.float64)
    P = k.DenseMatrix.from_numpy(ctx, p)
    P.device_ptr()
    v, gram = k.sliceRow(P, 100, 200), k.syrk(P)
    k.gatedStep(k.Gate.DECAY, k.fill(ctx, 2.0, 100, 64), k.fill(ctx, 1.0, 100, 64), v)
    assert np.array_equal(gram.to_numpy(), p.T @ p) and np.array_equal(v.to_numpy(), 2 * p[100:200] + 1)


@gpu
def test_operands_that_are_deferred_and_results_that_name_them(ctx):
    """Chains that are not computed yet as operands, and results in the operand's own handle."""
    import daphne_b200.kernels as k
    rng = np.random.default_rng(4)
    r, c = SHAPE
    a, b = rng.standard_normal(SHAPE), rng.standard_normal(SHAPE)
    off = np.array([[0], [100], [260]])
    M = lambda m: k.DenseMatrix.from_numpy(ctx, m)  # noqa: E731
    twice = lambda m: k.ewBinaryObjSca(k.BinaryOpCode.MUL, M(m), 2.0)  # noqa: E731
    s, d, ref = ctx.handle, int(k.Gate.DECAY), C.byref
    tok = rng.integers(0, r, (r, 1))
    w, h0 = rng.standard_normal((1, c)), rng.standard_normal((2, c))
    W, H0, OFF, T = M(w), M(h0), M(off), M(tok)
    none = lambda: C.c_void_p()  # noqa: E731
    calls = {
        "embed": (1, lambda o, x, y: lib.db2_embed(s, ref(o[0]), x.handle, T.handle, 1.0)),
        "embedGrad": (1, lambda o, x, y: lib.db2_embedGrad(s, ref(o[0]), x.handle, T.handle, r, 1.0, 0, 0)),
        "rmsNorm": (3, lambda o, x, y: lib.db2_rmsNorm(s, ref(o[0]), ref(o[1]), ref(o[2]), x.handle, y.handle, W.handle, 1e-6)),
        "rmsNormGrad": (2, lambda o, x, y: lib.db2_rmsNormGrad(s, ref(o[0]), ref(o[1]), x.handle, y.handle, W.handle, V.handle, x.handle)),
        "gatedScan": (2, lambda o, x, y: lib.db2_gatedScan(s, d, ref(o[0]), ref(o[1]), x.handle, y.handle, OFF.handle, H0.handle)),
        "gatedScanGrad": (3, lambda o, x, y: lib.db2_gatedScanGrad(s, d, ref(o[0]), ref(o[1]), ref(o[2]), x.handle, y.handle, y.handle,
                                                                 x.handle, OFF.handle, H0.handle, H0.handle)),
        "gatedStep": (2, lambda o, x, y: lib.db2_gatedStep(s, d, ref(o[0]), ref(o[1]), x.handle, y.handle, x.handle)),
    }
    V = M(np.abs(rng.standard_normal((r, 1))))
    for name, (n, call) in calls.items():
        def run(slots, x, y):
            check(call(slots, x, y))
            return [k.DenseMatrix(ctx, o).to_numpy() if own is None else own.to_numpy() for o, own in zip(slots, owners)]
        owners = [None] * n
        exp = run([none() for _ in range(n)], M(2 * a), M(2 * b))
        assert all(np.isfinite(e).all() for e in exp)
        got = run([none() for _ in range(n)], twice(a), twice(b))
        assert all(np.array_equal(e, q) for e, q in zip(exp, got)), name
        for i, e in enumerate(exp):  # every result of that shape in the place of either operand
            if e.shape != SHAPE:
                continue
            for which in (0, 1):
                x, y = twice(a), twice(b)
                keep = [k.ewBinaryObjSca(k.BinaryOpCode.ADD, m, 1.0) for m in (x, y)]
                owners = [None] * n
                owners[i] = (x, y)[which]
                slots = [none() for _ in range(n)]
                slots[i] = C.c_void_p(owners[i].handle.value)
                got = run(slots, x, y)
                assert all(np.array_equal(p, q) for p, q in zip(exp, got)), (name, i, which)
                assert np.array_equal(keep[0].to_numpy(), 2 * a + 1) and np.array_equal(keep[1].to_numpy(), 2 * b + 1), (name, i, which)


@gpu
def test_results_in_views_that_overlap_operands_are_refused(ctx):
    """A view is written where it lies.  Over the very elements of an operand that is allowed where the operator allows it;
    anything else that an operand or another result would share is refused, and nothing is written."""
    import daphne_b200.kernels as k
    rng = np.random.default_rng(6)
    p = rng.integers(-4, 5, (60, 20)).astype(np.float64)
    d, s, ref = int(k.Gate.DECAY), ctx.handle, C.byref
    M = lambda a: k.DenseMatrix.from_numpy(ctx, a)  # noqa: E731
    tok = M(rng.integers(0, 10, (10, 1)))
    slot = lambda m: C.c_void_p(m.handle.value)  # noqa: E731
    other = [M(rng.standard_normal((10, 8))) for _ in range(4)]
    v, st, w = M(np.ones((10, 1))), M(np.zeros((1, 8))), M(np.ones((1, 8)))
    o0, o1, o2, o3 = (m.handle for m in other)

    def calls(a):  # a: the operand; results by name, and whether they may be the operand itself
        z = a.handle
        return {
            "embed": lambda r: lib.db2_embed(s, ref(r), z, tok.handle, 1.0),
            "embedGrad": lambda r: lib.db2_embedGrad(s, ref(r), z, tok.handle, 10, 1.0, 0, 0),
            "embedGrad, added": lambda r: lib.db2_embedGrad(s, ref(r), z, tok.handle, 10, 1.0, 0, 1),
            "rmsNorm": lambda r: lib.db2_rmsNorm(s, ref(r), None, None, z, None, w.handle, 1e-6),
            "rmsNorm, sum": lambda r: lib.db2_rmsNorm(s, ref(C.c_void_p()), ref(r), None, o0, z, w.handle, 1e-6),
            "rmsNormGrad": lambda r: lib.db2_rmsNormGrad(s, ref(r), None, o0, z, w.handle, v.handle, None),
            "gatedScan": lambda r: lib.db2_gatedScan(s, d, ref(r), None, o0, z, None, None),
            "gatedScanGrad": lambda r: lib.db2_gatedScanGrad(s, d, ref(r), ref(C.c_void_p()), None, o0, None, z, o1, None, None, None),
            "gatedScanGrad, dx": lambda r: lib.db2_gatedScanGrad(s, d, ref(C.c_void_p()), ref(r), None, z, None, o2, o1, None, None, None),
            "gatedStep": lambda r: lib.db2_gatedStep(s, d, ref(r), ref(C.c_void_p()), z, o0, o1),
            "gatedStep, state": lambda r: lib.db2_gatedStep(s, d, ref(C.c_void_p()), ref(r), o0, z, r),
        }
    itself = {"rmsNorm", "rmsNorm, sum", "rmsNormGrad", "gatedScan", "gatedStep", "gatedStep, state"}
    for name in calls(other[0]):
        for rows, cols in ((0, 0), (3, 0), (0, 4), (9, 7), (5, -3), (10, 0), (0, 8), (40, 2)):
            P = M(p)
            P.device_ptr()
            a = k.sliceCol(k.sliceRow(P, 10, 20), 5, 13)
            r0, c0 = 10 + rows, 5 + cols
            r = k.sliceCol(k.sliceRow(P, r0, r0 + 10), c0, min(c0 + 8, 20)) if c0 + 8 <= 20 else None
            if r is None:
                continue
            apart = abs(rows) >= 10 or abs(cols) >= 8
            rc = calls(a)[name](slot(r))
            same = rows == 0 and cols == 0
            assert rc == (0 if apart or (same and name in itself) else 1), (name, rows, cols, rc)
            now = P.to_numpy()
            if rc:
                assert np.array_equal(now, p), (name, rows, cols)
            now[r0:r0 + 10, c0:c0 + 8] = p[r0:r0 + 10, c0:c0 + 8]
            assert np.array_equal(now, p), (name, rows, cols)
    P = M(p)
    P.device_ptr()
    a, b = k.sliceRow(P, 0, 10), k.sliceRow(P, 9, 19)
    g = M(rng.standard_normal((10, 20)))
    assert lib.db2_gatedStep(s, d, ref(slot(a)), ref(slot(b)), g.handle, g.handle, g.handle) == 1
    assert lib.db2_gatedStep(s, d, ref(slot(a)), ref(slot(k.sliceRow(P, 10, 20))), g.handle, g.handle, g.handle) == 0


@gpu
@pytest.mark.parametrize("update", ["step", "table gradient"])
@pytest.mark.parametrize("reader", ["none", "chain", "view", "sparse product"])
def test_updates_of_memory_that_a_caller_lent(ctx, update, reader):
    """A matrix that wraps a caller's device memory is updated there, whoever else reads it; what was asked for before keeps the
    values of that time."""
    import daphne_b200.kernels as k
    import torch
    rng = np.random.default_rng(8)
    p, g, x = (rng.integers(-4, 5, SHAPE).astype(np.float64) for _ in range(3))
    t = torch.as_tensor(p).cuda()
    torch.cuda.synchronize()
    P = k.DenseMatrix.wrap_device(ctx, t.data_ptr(), *SHAPE, SHAPE[1], np.float64, keep=t)
    M = lambda a: k.DenseMatrix.from_numpy(ctx, a)  # noqa: E731
    got, exp = None, 2 * p
    if reader == "chain":
        got = k.ewBinaryObjSca(k.BinaryOpCode.MUL, P, 2.0)
    elif reader == "view":
        got = k.sliceRow(P, 3, 7)
    elif reader == "sparse product":
        n = SHAPE[0]
        G = k.CSRMatrix.from_arrays(ctx, n, SHAPE[1], np.full(n, 2.0), np.zeros(n, dtype=np.uint64), np.arange(n + 1, dtype=np.uint64))
        got = k.ewMulCsrDense(G, P)
    if update == "step":
        k.gatedStep(k.Gate.DECAY, M(g), M(x), P)
        new = g * p + x
    else:
        tok, dy = rng.integers(0, SHAPE[0], (40, 1)), rng.integers(-4, 5, (40, SHAPE[1])).astype(np.float64)
        k.embedGrad(M(dy), M(tok), SHAPE[0], add_to=P)
        new = p.copy()
        np.add.at(new, tok[:, 0], dy)
    ctx.sync()
    assert np.array_equal(t.cpu().numpy(), new) and np.array_equal(P.to_numpy(), new)
    if reader == "chain":
        assert np.array_equal(got.to_numpy(), exp)
    elif reader == "view":
        assert np.array_equal(got.to_numpy(), new[3:7])
    elif reader == "sparse product":
        assert np.array_equal(k.aggRowCsr(k.AggOpCode.SUM, got).to_numpy()[:, 0], exp[:, 0])


@gpu
def test_a_table_gradient_added_to_its_own_operand(ctx):
    """The rows are read before they are added to, also where the memory is a caller's: the matrix then moves."""
    import daphne_b200.kernels as k
    import torch
    rng = np.random.default_rng(9)
    p, tok = rng.integers(-4, 5, (50, 30)).astype(np.float64), rng.integers(0, 50, (50, 1))
    exp = p.copy()
    np.add.at(exp, tok[:, 0], p)
    t = torch.as_tensor(p).cuda()
    torch.cuda.synchronize()
    for P in (k.DenseMatrix.from_numpy(ctx, p), k.DenseMatrix.wrap_device(ctx, t.data_ptr(), 50, 30, 30, np.float64, keep=t)):
        k.embedGrad(P, k.DenseMatrix.from_numpy(ctx, tok), 50, add_to=P)
        assert np.array_equal(P.to_numpy(), exp)
