"""Matrices of 16-bit and 8-bit floating-point types: casts (one rounding to nearest even, bit for bit), views, fill and
transfers, and the refusals of the operators that do not take them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SPECIAL = [0.0, -0.0, 1.0, 1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -9, 1.0 + 2.0 ** -11, 65504.0, 65520.0, 1e5, 3.4e38, 2.0 ** -24,
           2.0 ** -25, 1e-40, np.inf, -np.inf, np.nan]


def _bits(x, t):
    """numpy values -> bit patterns in torch type t (one rounding)."""
    return torch.as_tensor(x).to(t).view(torch.int16).numpy().view(np.uint16)


@pytest.mark.parametrize("src", [np.float64, np.float32])
@pytest.mark.parametrize("name,t", [("float16", torch.float16), ("bfloat16", torch.bfloat16)])
def test_casts_round_once_to_nearest_even(ctx, src, name, t):
    import daphne_b200.kernels as k
    rng = np.random.default_rng(1)
    # singles are doubles, too: every rounding shows on them, and a double may not be rounded to a single first
    x = np.concatenate([SPECIAL, rng.standard_normal(500) * 10.0 ** rng.integers(-9, 9, 500)]).astype(np.float32).astype(src)
    x = x.reshape(-1, 4)
    code = np.float16 if name == "float16" else k.BFLOAT16
    h = k.castObj(k.DenseMatrix.from_numpy(ctx, x), code)
    got = h.to_numpy()
    exp = _bits(x.astype(np.float32), t)
    nan = np.isnan(x)
    assert np.array_equal(got.view(np.uint16)[~nan], exp[~nan])
    back = k.castObj(h, src).to_numpy()
    wide = torch.as_tensor(exp.view(np.int16)).view(t).to(torch.float64).numpy()
    assert back.dtype == src and np.array_equal(back[~nan], wide[~nan]) and np.isnan(back[nan]).all()
    part = k.castObj(k.sliceCol(k.sliceRow(h, 3, 50), 1, 3), np.float64).to_numpy()
    assert np.array_equal(part, wide[3:50, 1:3], equal_nan=True)


def test_a_double_next_to_a_tie_is_rounded_once(ctx):
    import daphne_b200.kernels as k
    x = np.array([[1.0 + 2.0 ** -8 + 2.0 ** -40, 1.0 + 2.0 ** -11 + 2.0 ** -40]])
    b = k.castObj(k.castObj(k.DenseMatrix.from_numpy(ctx, x), k.BFLOAT16), np.float64).to_numpy()
    h = k.castObj(k.castObj(k.DenseMatrix.from_numpy(ctx, x), np.float16), np.float64).to_numpy()
    assert b[0, 0] == 1.0 + 2.0 ** -7 and h[0, 1] == 1.0 + 2.0 ** -10


def test_eight_bit_values_widen_exactly(ctx):
    import daphne_b200.kernels as k
    bits = np.arange(256, dtype=np.uint8).reshape(16, 16)
    d = torch.as_tensor(bits).cuda()
    m = k.DenseMatrix.wrap_device(ctx, d.data_ptr(), 16, 16, 16, k.FLOAT8_E4M3, keep=d)
    torch.cuda.synchronize()
    exp = torch.as_tensor(bits).view(torch.float8_e4m3fn).double().numpy()
    for t in (np.float64, np.float32):
        assert np.array_equal(k.castObj(m, t).to_numpy(), exp.astype(t), equal_nan=True)
    assert np.array_equal(m.to_numpy(), bits)


def test_fill_and_host_round_trip(ctx):
    import daphne_b200.kernels as k
    assert np.array_equal(k.fill(ctx, 1.5, 7, 9, dtype=np.float16).to_numpy(), np.full((7, 9), 1.5, dtype=np.float16))
    a = np.random.default_rng(2).standard_normal((30, 11)).astype(np.float16)
    m = k.DenseMatrix.from_numpy(ctx, a)
    m.device_ptr()
    assert np.array_equal(m.to_numpy(), a) and np.array_equal(k.sliceCol(m, 2, 5).to_numpy(), a[:, 2:5])


def test_operators_without_these_types_refuse_them(ctx, tmp_path):
    import daphne_b200.kernels as k
    A, B, U = k.AggOpCode, k.BinaryOpCode, k.UnaryOpCode
    for dtype in (np.float16, k.BFLOAT16, k.FLOAT8_E4M3):
        m = k.DenseMatrix.empty(ctx, 8, 8, dtype, zero=True)
        for call in (lambda: k.ewBinaryMat(B.ADD, m, m), lambda: k.ewBinaryObjSca(B.MUL, m, 1), lambda: k.ewUnaryMat(U.ABS, m),
                     lambda: k.aggRow(A.SUM, m), lambda: k.aggCol(A.SUM, m), lambda: k.aggAll(A.SUM, m),
                     lambda: k.matMul(m, m), lambda: k.syrk(m), lambda: k.gemv(m, m), lambda: k.solve(m, m),
                     lambda: k.transpose(m), lambda: k.aggCum(A.SUM, m), lambda: k.colBind(m, m),
                     lambda: k.diagMatrix(k.sliceCol(m, 0, 1)), lambda: k.writeDaphne(m, tmp_path / "x.dbdf"),
                     lambda: k.cond(m, m, m) if dtype == np.float16 else k.transpose(m)):
            with pytest.raises(k.Db2Error) as e:
                call()
            assert e.value.code == 4, e.value
