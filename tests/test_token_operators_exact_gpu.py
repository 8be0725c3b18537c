"""What the operators on sequences of tokens are to give exactly, or to a few roundings whatever the size of the arguments."""
import numpy as np
import pytest
import torch

from daphne_b200 import lib as names
from daphne_b200.lib import check, lib
from tests.seq_util import TYPES, Mat, stream

gpu = pytest.mark.gpu


def _eight_bits(tname, s, w, group, eps=1e-5):
    t, code = TYPES[tname]
    rows, cols = s.shape
    S, W = Mat(s, t), Mat(w, t) if w is not None else None
    width = group or cols
    n = -(-cols // width)
    Y, Q = Mat(torch.zeros(rows, cols), torch.uint8), Mat.empty(rows, n, torch.float32)
    check(lib.db2k_rms_norm_q8(code, *S.at[:1], rows, cols, S.ld, None, 0, W.ptr if W else None, eps, None, 0, *Y.at, *Q.at,
                               group, None, stream()))
    # 1 / rms is common to a row: a group's values are those of s * weight over their largest, times 448
    p = S.f64() * (W.f64() if W else 1.0)
    full = np.zeros((rows, n * width))
    full[:, :cols] = np.abs(p)
    most = np.repeat(full.reshape(rows, n, width).max(2), width, 1)[:, :cols]
    with np.errstate(invalid="ignore"):
        return Y, Q, p * 448.0 / np.where(most == 0, 1.0, most)


@gpu
@pytest.mark.parametrize("tname,weighted", [("bf16", True), ("bf16", False), ("f16", False), ("f32", False)])
@pytest.mark.parametrize("group", [0, 16, 128, 512])
@pytest.mark.parametrize("rows,cols", [(3, 7), (300, 33), (64, 1024), (200, 130), (2, 40000), (5, 16501), (160, 5120)])
def test_eight_bit_results_are_the_nearest_values(tname, weighted, group, rows, cols):
    """Products of two bf16 values (16 bits) and their quotients' ties are exact in 64 bits, and so are those of short single
    values: a tie goes to the even neighbour, every other quotient to the nearest value."""
    rng = np.random.default_rng(rows + cols)
    s = rng.integers(-255, 256, (rows, cols)) * 2.0 ** rng.integers(-9, 1, (rows, cols))
    s[0] = 0
    if rows > 1:
        s[1] = rng.integers(-31, 32, cols)  # most quotients with 28 are ties or representable
        s[1, ::16] = 28
    w = rng.integers(128, 256, (1, cols)) * 2.0 ** -7 if weighted else None
    Y, Q, q = _eight_bits(tname, s, w, group)
    exp = torch.as_tensor(q).float().to(torch.float8_e4m3fn).view(torch.uint8)
    got = Y.view.cpu()
    zero = torch.as_tensor(q == 0)
    assert torch.equal(got[~zero], exp[~zero]) and bool(((got[zero] & 0x7f) == 0).all())
    assert Y.guards_intact() and Q.guards_intact()


@gpu
def test_eight_bit_scales_far_from_one():
    """Rows whose root mean square is far from one, the smallest scales, and groups with an infinity."""
    rng = np.random.default_rng(1)
    for size in (1e-15, 1e-6, 1e6, 1e15):
        s = rng.standard_normal((4, 96)) * size
        Y, Q, q = _eight_bits("bf16", s, rng.standard_normal((1, 96)), 32, 0.0)
        assert torch.equal(Y.view.cpu(), torch.as_tensor(q).float().to(torch.float8_e4m3fn).view(torch.uint8))
    w = np.ones((1, 64))
    w[0, 5] = np.inf
    w[0, 40] = 3e38
    Y, Q, _ = _eight_bits("f32", np.ones((2, 64)), w, 32, 0.0)
    v = Y.view.cpu().view(torch.float8_e4m3fn).double().numpy()
    assert np.isinf(Q.f64()[:, 0]).all() and np.isnan(v[:, 5]).all() and not np.delete(v[:, :32], 5, 1).any()
    assert (v[:, 40] == 448).all() and not np.delete(v[:, 32:], 8, 1).any() and np.isfinite(Q.f64()[:, 1]).all()
    # y below 448 times the smallest normal number: the scale stays there, the quotient is by it
    s = np.zeros((1, 32))
    s[0, :4] = [1.0, -0.5, 2.0 ** -5, 1.5]
    w = np.full((1, 32), 2.0 ** -126)
    Y, Q, _ = _eight_bits("f32", s, w, 32, 1.0)
    y = (s / np.sqrt((s * s).mean() + 1.0))[0, :4]
    v = Y.view.cpu().view(torch.float8_e4m3fn).double().numpy()[0]
    assert Q.f64()[0, 0] == 2.0 ** -126 and (np.abs(v[:4] - y) <= np.abs(y) * 2.0 ** -4).all() and not v[4:].any()


def _gate_values(tname, g):
    """f and 1 - f as the kernels have them: steps from a state of one without an input, and from none with an input of one."""
    t, code = TYPES[tname]
    G, n = Mat(g, t), g.shape[1]
    out = []
    for state in (1.0, 0.0):
        X, S, N = Mat(torch.full((1, n), 1.0 - state), t), Mat(torch.full((1, n), state), torch.float32), Mat.empty(1, n, torch.float32)
        check(lib.db2k_gated_step(code, names.GATE_SIGMOID, *G.at, *X.at, 1, n, *S.at, *N.at, None, 0, stream()))
        out.append(N.f64()[0])
    return G.f64()[0], *out


@gpu
@pytest.mark.parametrize("tname", ["f32", "f16", "bf16"])
def test_sigmoid_is_as_accurate_for_large_arguments_as_for_small_ones(tname):
    """Half steps (2^-24) that the parts of e = exp(-g), f = 1 / (1 + e) and 1 - f = e f may be off by: the base-2
    exponential 2^-22.5, so 2.9; its correction 1; 1 + e 1; the reciprocal (a unit) 2; the last product 1; the sums and
    products of the step round nothing.  One more for all second-order terms: 9."""
    rng = np.random.default_rng(2)
    g = np.concatenate([rng.uniform(-86, 86, 20000), rng.standard_normal(5000) * 2, np.linspace(-86, 86, 173), [0.0, -0.0]])
    g, f, o = _gate_values(tname, g[None, :])
    ef, eo = 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))
    assert (np.abs(f - ef) <= 9 * 2.0 ** -24 * ef).all(), np.max(np.abs(f - ef) / ef) * 2 ** 24
    assert (np.abs(o - eo) <= 9 * 2.0 ** -24 * eo).all(), np.max(np.abs(o - eo) / eo) * 2 ** 24
    # the ends: f stays at 2^-125 and above, 1 - f becomes zero, and nothing else happens there
    g, f, o = _gate_values(tname, np.array([[-86.7, -90.0, -1e3, -6e4, -np.inf, 88.0, 150.0, 1e3, 6e4, np.inf, np.nan]]))
    assert (f[:5] >= 2.0 ** -125).all() and (f[:5] <= 2.0 ** -124).all() and (o[:5] == 1).all()
    assert (f[5:10] == 1).all() and (o[5:10] <= 2.0 ** -125).all() and (o[5:10] >= 0).all()
    assert np.isnan(f[10]) and np.isnan(o[10])


@gpu
@pytest.mark.parametrize("src", ["float16", "bfloat16", "float8_e4m3"])
@pytest.mark.parametrize("dst", ["float16", "bfloat16"])
def test_casts_between_the_short_types(ctx, src, dst):
    """Every bit pattern of the source, rounded once to nearest even; a cast to the type itself is a copy."""
    import daphne_b200.kernels as k
    t = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float8_e4m3": torch.float8_e4m3fn}
    code = {"float16": np.float16, "bfloat16": k.BFLOAT16, "float8_e4m3": k.FLOAT8_E4M3}
    bits = torch.arange(256 if src == "float8_e4m3" else 65536).to(torch.uint8 if src == "float8_e4m3" else torch.int32)
    bits = bits.view(-1, 64) if src == "float8_e4m3" else bits.to(torch.int16).view(-1, 64)
    d = bits.cuda()
    m = k.DenseMatrix.wrap_device(ctx, d.data_ptr(), d.shape[0], 64, 64, code[src], keep=d)
    torch.cuda.synchronize()
    got = k.castObj(k.sliceCol(m, 1, 64), code[dst]).to_numpy().view(np.int16)
    x = bits[:, 1:].contiguous().view(t[src])
    exp = x.to(t[dst])
    nan = x.float().isnan()
    assert torch.equal(torch.as_tensor(got.copy())[~nan], exp.view(torch.int16)[~nan])
    assert bool(torch.as_tensor(got.copy()).view(t[dst]).float()[nan].isnan().all())
