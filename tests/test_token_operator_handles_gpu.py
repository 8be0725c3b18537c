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
