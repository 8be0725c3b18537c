"""The token operators together, as a model uses them: embedding -> norm -> products -> gated recurrence -> norm with the
embedding as the residual, its gradients (against automatic differentiation of the formulas in 64 bits on the CPU), and
the same model fed token by token."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

V, C, EPS = 23, 24, 1e-6
OFF = [0, 7, 7, 40, 61]


def _params(seed):
    rng = np.random.default_rng(seed)
    p = {"E": rng.standard_normal((V, C)) * 0.3, "w1": 1 + 0.2 * rng.standard_normal((1, C)),
         "w2": 1 + 0.2 * rng.standard_normal((1, C)), "Wg": rng.standard_normal((C, C)) / np.sqrt(C),
         "Wx": rng.standard_normal((C, C)) / np.sqrt(C), "h0": rng.standard_normal((len(OFF) - 1, C))}
    tok = rng.integers(-1, V, (OFF[-1], 1))
    return p, tok, rng.standard_normal((OFF[-1], C)), rng.standard_normal((len(OFF) - 1, C))


def _reference(p, tok, c, cl):
    t = {k: torch.tensor(v, requires_grad=True) for k, v in p.items()}
    tok = torch.as_tensor(tok[:, 0])

    def norm(s, w):
        return s * torch.rsqrt((s * s).mean(1, keepdim=True) + EPS) * w
    e = torch.where((tok >= 0)[:, None], t["E"][tok.clamp(min=0)] * C ** 0.5, 0.0)
    n = norm(e, t["w1"])
    f, x = torch.sigmoid(n @ t["Wg"]), n @ t["Wx"]
    rows, lasts = [], []
    for s in range(len(OFF) - 1):
        v = t["h0"][s]
        for r in range(OFF[s], OFF[s + 1]):
            v = f[r] * v + (1 - f[r]) * x[r]
            rows.append(v)
        lasts.append(v)
    y = norm(torch.stack(rows) + e, t["w2"])
    ((y * torch.as_tensor(c)).sum() + (torch.stack(lasts) * torch.as_tensor(cl)).sum()).backward()
    return y.detach().numpy(), {k: v.grad.numpy() for k, v in t.items()}


def test_a_training_step_and_decoding(ctx):
    import daphne_b200.kernels as k
    p, tok, c, cl = _params(1)
    M = lambda a: k.DenseMatrix.from_numpy(ctx, np.ascontiguousarray(a))  # noqa: E731
    m = {n: M(v) for n, v in p.items()}
    T, off, scale, gate = M(tok), M(np.array(OFF).reshape(-1, 1)), C ** 0.5, k.Gate.SIGMOID
    e = k.embed(m["E"], T, scale)
    n, _, r1 = k.rmsNorm(e, m["w1"], EPS)
    g, x = k.matMul(n, m["Wg"]), k.matMul(n, m["Wx"])
    h, last = k.gatedScan(gate, g, x, off, m["h0"])
    y, s, r2 = k.rmsNorm(h, m["w2"], EPS, residual=e)
    ds, dw2 = k.rmsNormGrad(M(c), s, r2, m["w2"])
    dg, dx, dh0 = k.gatedScanGrad(gate, g, x, h, ds, off, m["h0"], M(cl))
    dn = k.ewBinaryMat(k.BinaryOpCode.ADD, k.matMul(dg, m["Wg"], transb=True), k.matMul(dx, m["Wx"], transb=True))
    de, dw1 = k.rmsNormGrad(dn, e, r1, m["w1"], dsum=ds)
    got = {"E": k.embedGrad(de, T, V, scale), "w1": dw1, "w2": dw2, "Wg": k.matMul(n, dg, transa=True),
           "Wx": k.matMul(n, dx, transa=True), "h0": dh0}
    yr, gr = _reference(p, tok, c, cl)
    # padding rows are zeros: 1 / rms is 1000 there, and the rounding errors of its neighbours grow with it
    np.testing.assert_allclose(y.to_numpy(), yr, rtol=0, atol=1e-11)
    for name, ref in gr.items():
        np.testing.assert_allclose(got[name].to_numpy(), ref, rtol=0, atol=1e-10 * max(1.0, np.abs(ref).max()), err_msg=name)
    # token by token: one row per sequence and call, states updated in place
    out = y.to_numpy()
    lens = np.diff(OFF)
    state = M(p["h0"])
    for t in range(lens.max()):
        live = np.flatnonzero(lens > t)
        now = M(tok[[OFF[i] + t for i in live]])
        rows = M(state.to_numpy()[live])
        e1 = k.embed(m["E"], now, scale)
        n1, _, _ = k.rmsNorm(e1, m["w1"], EPS)
        h1 = k.gatedStep(gate, k.matMul(n1, m["Wg"]), k.matMul(n1, m["Wx"]), rows)
        y1 = k.rmsNorm(h1, m["w2"], EPS, residual=e1)[0].to_numpy()
        np.testing.assert_allclose(y1, out[[OFF[i] + t for i in live]], rtol=0, atol=1e-11)
        new = state.to_numpy()
        new[live] = rows.to_numpy()
        state = M(new)
    np.testing.assert_allclose(state.to_numpy(), last.to_numpy(), rtol=0, atol=1e-12)


def test_the_same_step_in_sixteen_bits(ctx):
    """bf16 storage with float states: every stored value is rounded once (2^-8 relative); four roundings in a row lie
    between the table and the result, and the last norm divides by a root mean square of about one."""
    import daphne_b200.kernels as k
    p, tok, c, cl = _params(2)
    tok = np.maximum(tok, 0)
    yr, _ = _reference(p, tok, c, cl)
    B = lambda a: k.castObj(k.DenseMatrix.from_numpy(ctx, np.ascontiguousarray(a)), k.BFLOAT16)  # noqa: E731
    F = lambda a: k.DenseMatrix.from_numpy(ctx, np.ascontiguousarray(a, dtype=np.float32))  # noqa: E731
    T, off = k.DenseMatrix.from_numpy(ctx, tok), k.DenseMatrix.from_numpy(ctx, np.array(OFF).reshape(-1, 1))
    e = k.embed(B(p["E"]), T, C ** 0.5)
    n, _, _ = k.rmsNorm(e, B(p["w1"]), EPS)
    n32 = k.castObj(n, np.float32)
    g, x = (k.castObj(k.matMul(n32, F(p[w])), k.BFLOAT16) for w in ("Wg", "Wx"))
    h, _ = k.gatedScan(k.Gate.SIGMOID, g, x, off, F(p["h0"]))
    y, _, _ = k.rmsNorm(h, B(p["w2"]), EPS, residual=e)
    got = k.castObj(y, np.float64).to_numpy()
    # table, weights, n, g, x, h, s, w2, y: nine roundings of 2^-8 on values of up to 4, gates pass on a quarter of g's
    assert np.abs(got - yr).max() < 9 * 4 * 2.0 ** -8
    q, sc, _, _ = k.rmsNormQ8(h, B(p["w2"]), EPS, residual=e, group=16)
    deq = k.castObj(q, np.float64).to_numpy() * np.repeat(sc.to_numpy().astype(np.float64), 16, 1)[:, :C]
    assert (np.abs(deq - got) <= np.abs(got) * (2.0 ** -4 + 2.0 ** -7) + np.repeat(sc.to_numpy(), 16, 1)[:, :C] * 2.0 ** -9).all()
