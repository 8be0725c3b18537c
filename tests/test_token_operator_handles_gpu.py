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
