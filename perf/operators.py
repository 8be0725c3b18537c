"""Operators of a recurrent sequence model, as they are measured: embedding lookup and its gradient, root-mean-square
norm with the residual's addition (also with an 8-bit output), gated linear recurrence over packed sequences with its
gradient and its single-token step.

Where `own` is false, run() computes them in elementary torch operations, in 32 bits (64 for doubles); where it is true
it makes the framework's calls on the same buffers."""
import math

import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # one new token for each of four requests that are being answered: latency
        {"name": "embed_four_tokens", "op": "embed", "type": "bf16", "rows": 4, "cols": 1024, "vocab": 32000, "pad": 0.0},
        # a batch of prompts entering a model with a large vocabulary
        {"name": "embed_prompts", "op": "embed", "type": "bf16", "rows": 16384, "cols": 4096, "vocab": 128256, "pad": 0.02},
        # training batch: the gradient of the whole table, tokens as frequent as words are
        {"name": "embed_grad_batch", "op": "embed_grad", "type": "bf16", "rows": 16384, "cols": 2048, "vocab": 64000, "pad": 0.02},
        # a small categorical model in single precision with odd sizes
        {"name": "embed_grad_odd", "op": "embed_grad", "type": "f32", "rows": 5001, "cols": 515, "vocab": 3011, "pad": 0.0},
        # one new token for each of eight requests: latency
        {"name": "norm_eight_rows", "op": "norm", "type": "bf16", "rows": 8, "cols": 4096, "residual": True},
        # training: forward and backward over a batch
        {"name": "norm_train_batch", "op": "norm_train", "type": "bf16", "rows": 16384, "cols": 4096, "residual": True},
        # prompts entering an 8-bit product: one scale for 128 columns
        {"name": "norm_q8_prompts", "op": "norm_q8", "type": "bf16", "rows": 8192, "cols": 5120, "residual": True, "group": 128},
        # doubles of a data analysis script, odd width, no residual, with the gradient
        {"name": "norm_train_double", "op": "norm_train", "type": "f64", "rows": 10007, "cols": 333, "residual": False},
        # one new token for each of 64 requests: latency
        {"name": "step_64_requests", "op": "step", "type": "bf16", "rows": 64, "cols": 2048, "gate": "sigmoid"},
        # prompts of different lengths packed into one batch, with padding rows behind the last one
        {"name": "scan_ragged_prompts", "op": "scan", "type": "f16", "rows": 30000, "cols": 2560, "gate": "sigmoid", "seqs": 37, "ragged": True},
        # one long series of few channels in single precision, such as measurements
        {"name": "scan_long_series", "op": "scan", "type": "f32", "rows": 100000, "cols": 96, "gate": "decay", "seqs": 1, "ragged": False},
        # training: forward and backward over a batch of equally long sequences
        {"name": "scan_train_batch", "op": "scan_train", "type": "bf16", "rows": 32768, "cols": 2048, "gate": "sigmoid", "seqs": 8, "ragged": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "norm", "norm_q8", "norm_train", "step", "scan", "scan_train"])
    types = ["bf16", "f16", "f32"] if op == "norm_q8" else ["bf16", "f16", "f32", "f64"]
    c = {"op": op, "type": rng.choice(types)}
    c["cols"] = _log(rng, 1, 8192)
    most = (1 << 25) // c["cols"]
    c["rows"] = _log(rng, 1, min(512 if op == "step" else 40000, most))
    if op.startswith("embed"):
        c["vocab"] = _log(rng, 16, min(130000, max(16, (1 << 27) // c["cols"])))
        c["pad"] = rng.choice([0.0, 0.1])
    elif op.startswith("norm"):
        c["residual"] = rng.random() < 0.6
        if op == "norm_q8":
            c["group"] = rng.choice([0, 32, 64, 128, 256])
    else:
        c["gate"] = rng.choice(["decay", "sigmoid"])
        if op != "step":
            c["seqs"] = _log(rng, 1, min(64, c["rows"]))
            c["ragged"] = rng.random() < 0.5
            if not c["ragged"]:
                c["rows"] -= c["rows"] % c["seqs"]
    return c


def _wide(t):
    """The type that a plain form computes in."""
    return torch.float64 if t == torch.float64 else torch.float32


def _normal(rows, cols, t, gen, mean=0.0, sd=1.0):
    x = torch.empty(rows, cols, dtype=_wide(t), device="cuda").normal_(mean, sd, generator=gen)
    return x.to(t)


def _lengths(case, seed):
    """Rows of every sequence: equal ones, or ragged ones (an empty one among three and more) with rows left over at the end."""
    n, rows = case["seqs"], case["rows"]
    if not case["ragged"]:
        return [rows // n] * n
    gen = torch.Generator().manual_seed(seed + 1)
    used = rows - rows // 50
    share = torch.rand(n, generator=gen, dtype=torch.float64) ** 2 + 0.02
    if n >= 3:
        share[n // 2] = 0.0
    cum = torch.cumsum(share, 0) / share.sum() * used
    ends = [int(v) for v in cum.floor().tolist()]
    ends[-1] = used
    return [b - a for a, b in zip([0] + ends[:-1], ends)]


def prepare(case, seed):
    t, rows, cols, op = TYPES[case["type"]], case["rows"], case["cols"], case["op"]
    wide = _wide(t)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    empty = lambda r, c, ty: torch.zeros(r, c, dtype=ty, device="cuda")  # noqa: E731
    s = {"case": dict(case)}
    if op.startswith("embed"):
        v = case["vocab"]
        # word frequencies fall with the rank; the ranks lie anywhere in the table
        rank = torch.exp(torch.rand(rows, dtype=torch.float64, device="cuda", generator=gen) * math.log(v)).long().clamp(1, v) - 1
        place = torch.randperm(v, device="cuda", generator=gen)
        tok = place[rank]
        pad = torch.rand(rows, device="cuda", generator=gen) < case["pad"]
        s["tokens"] = torch.where(pad, torch.full_like(tok, -1), tok)
        s["scale"] = math.sqrt(cols)
        if op == "embed":
            s["table"] = _normal(v, cols, t, gen, 0.0, 0.02)
            s["res"] = empty(rows, cols, t)
        else:
            s["grad"] = _normal(rows, cols, t, gen)
            s["res"] = empty(v, cols, t)
    elif op.startswith("norm"):
        s["x"] = _normal(rows, cols, t, gen)
        s["residual"] = _normal(rows, cols, t, gen, 0.1, 3.0) if case["residual"] else None
        s["weight"] = _normal(1, cols, t, gen, 1.0, 0.2)
        s["sum"] = empty(rows, cols, t) if case["residual"] else None
        s["rstd"] = empty(rows, 1, wide)
        s["res"] = empty(rows, cols, torch.float8_e4m3fn if op == "norm_q8" else t)
        if op == "norm_q8":
            s["scales"] = empty(rows, -(-cols // case["group"]) if case["group"] else 1, torch.float32)
        if op == "norm_train":
            s["grad"] = _normal(rows, cols, t, gen)
            s["dsum"] = _normal(rows, cols, t, gen) if case["residual"] else None
            s["dx"], s["dweight"] = empty(rows, cols, t), empty(1, cols, wide)
    else:
        if case["gate"] == "sigmoid":
            s["g"] = _normal(rows, cols, t, gen, 2.0, 2.0)
        else:
            s["g"] = torch.exp(-0.2 * torch.rand(rows, cols, dtype=wide, device="cuda", generator=gen) ** 2).to(t)
        s["x"] = _normal(rows, cols, t, gen)
        s["h"] = empty(rows, cols, t)
        if op == "step":
            s["state"], s["new_state"] = _normal(rows, cols, wide, gen), empty(rows, cols, wide)
        else:
            lengths = _lengths(case, seed)
            n, s["longest"] = len(lengths), max(lengths)
            # equally long sequences need no offsets
            s["offsets"] = torch.tensor([0] + lengths).cumsum(0).cuda() if case["ragged"] else None
            s["h0"], s["last"] = _normal(n, cols, wide, gen), empty(n, cols, wide)
            if op == "scan_train":
                s["grad"], s["grad_last"] = _normal(rows, cols, t, gen), _normal(n, cols, wide, gen)
                s["dg"], s["dx"], s["dh0"] = empty(rows, cols, t), empty(rows, cols, t), empty(n, cols, wide)
    if own:
        s["scratch"] = _scratch(s)
    return s


def work(case):
    t, rows, cols, op = TYPES[case["type"]], case["rows"], case["cols"], case["op"]
    e, w = t.itemsize, _wide(t).itemsize
    n = rows * cols
    if op == "embed":
        distinct = min(rows, case["vocab"])
        return {"bytes": n * e + distinct * cols * e + 8 * rows, "flops": n}
    if op == "embed_grad":
        return {"bytes": n * e + case["vocab"] * cols * e + 8 * rows, "flops": n}
    if op.startswith("norm"):
        moved = n * e * (3 if case["residual"] else 1) + cols * e + rows * w  # inputs, the sum, the weights, the statistics
        if op == "norm_q8":
            return {"bytes": moved + n + 4 * rows * (-(-cols // case["group"]) if case["group"] else 1), "flops": 6 * n}
        moved += n * e
        if op == "norm_train":  # the gradients, the sum again
            return {"bytes": moved + n * e * (4 if case["residual"] else 3) + cols * (e + w) + rows * w, "flops": 16 * n}
        return {"bytes": moved, "flops": 5 * n}
    if op == "step":
        return {"bytes": n * (3 * e + 2 * w), "flops": 8 * n}
    states = case["seqs"] * cols * w
    if op == "scan":
        return {"bytes": 3 * n * e + 2 * states, "flops": 8 * n}
    reads = 4 if case["gate"] == "sigmoid" else 3
    return {"bytes": 3 * n * e + 2 * states + (reads + 2) * n * e + 3 * states, "flops": 20 * n}


# ---- plain forms ----

def _plain_embed(s):
    tok, table = s["tokens"], s["table"]
    y = table[tok.clamp(min=0)].to(_wide(table.dtype)) * s["scale"]
    return (y * (tok >= 0)[:, None]).to(table.dtype)


def _plain_embed_grad(s):
    tok, grad, v = s["tokens"], s["grad"], s["case"]["vocab"]
    sums = torch.zeros(v + 1, grad.shape[1], dtype=_wide(grad.dtype), device="cuda")  # the last row takes the padding
    sums.index_add_(0, torch.where(tok < 0, v, tok), grad.to(sums.dtype))
    return (sums[:v] * s["scale"]).to(grad.dtype)


def _plain_norm(s):
    """(the sum as it is stored, in the wide type; 1 / rms; the normalised and weighted values, not rounded)"""
    x = s["x"]
    wide = _wide(x.dtype)
    v = x.to(wide)
    if s["residual"] is not None:
        v = (v + s["residual"].to(wide)).to(x.dtype).to(wide)
    rstd = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
    return v, rstd, v * rstd * s["weight"].to(wide)


def _plain_q8(y, group):
    rows, cols = y.shape
    group = group or cols
    full = torch.zeros(rows, -(-cols // group) * group, dtype=y.dtype, device="cuda")
    full[:, :cols] = y
    full = full.view(rows, -1, group)
    most = full.abs().amax(2)
    scales = torch.where(most > 0, most / E4M3_MAX, torch.ones_like(most))
    return (full / scales[:, :, None]).view(rows, -1)[:, :cols].to(torch.float8_e4m3fn), scales


def _plain_norm_grad(s, v, rstd):
    wide = v.dtype
    grad = s["grad"].to(wide)
    t = grad * s["weight"].to(wide)
    dx = rstd * (t - v * rstd * rstd * (t * v).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].to(wide)
    return dx.to(s["x"].dtype), (grad * v * rstd).sum(0, keepdim=True)


def _plain_scan(f, u, longest):
    """h[t] = f[t] h[t-1] + u[t] down the rows by doubling the span: a row takes in the row a span above it. A sequence's
    first row has f = 0, so that nothing reaches into it."""
    f, u, span = f.clone(), u.clone(), 1
    while span < longest:
        head = u[span:] + f[span:] * u[:-span]
        f[span:] = f[span:] * f[:-span]
        u[span:] = head
        span *= 2
    return u


def _plain_gates(s):
    g, x = s["g"].to(_wide(s["g"].dtype)), s["x"].to(_wide(s["g"].dtype))
    if s["case"]["gate"] == "decay":
        return g, x, x
    f = torch.sigmoid(g)
    return f, torch.sigmoid(-g) * x, x


def _plain_sequences(s):
    """(first row of every sequence, the row behind its last, which of them have rows)"""
    n, rows = s["case"]["seqs"], s["case"]["rows"]
    off = s["offsets"] if s["offsets"] is not None else torch.arange(n + 1, device="cuda") * (rows // n)
    return off[:-1], off[1:], off[1:] > off[:-1]


def _plain_scan_forward(s):
    f, u, x = _plain_gates(s)
    rows = s["case"]["rows"]
    first, end, some = _plain_sequences(s)
    # states enter by the first rows: empty sequences write to a row behind the last
    at = torch.where(some, first, rows)
    into = torch.zeros(rows + 1, f.shape[1], dtype=f.dtype, device="cuda")
    into[at] = s["h0"]
    starts = torch.zeros(rows + 1, dtype=torch.bool, device="cuda")
    starts[at] = True
    starts = starts[:rows, None]
    h = _plain_scan(torch.where(starts, 0.0, f), u + f * into[:rows], s["longest"])
    inside = (torch.arange(rows, device="cuda") < end[-1])[:, None]
    h = torch.where(inside, h, 0.0)
    last = torch.where(some[:, None], h[(end - 1).clamp(min=0)], s["h0"])
    return f, x, h, last, starts, into[:rows], inside


def _plain_scan_grad(s, f, x, h, starts, into, inside):
    rows = f.shape[0]
    first, end, some = _plain_sequences(s)
    above = torch.where(starts, into, torch.cat([torch.zeros_like(h[:1]), h[:-1]]))
    at = torch.where(some, (end - 1).clamp(min=0), rows)
    entering = torch.zeros(rows + 1, f.shape[1], dtype=f.dtype, device="cuda")
    entering[at] = s["grad_last"]
    ends = torch.zeros(rows + 1, dtype=torch.bool, device="cuda")
    ends[at] = True
    # delta[t] = grad[t] + f[t+1] delta[t+1], from the last row up
    below = torch.where(ends[:rows, None], 0.0, torch.cat([f[1:], torch.zeros_like(f[:1])]))
    delta = _plain_scan(below.flip(0), (s["grad"].to(f.dtype) + entering[:rows]).flip(0), s["longest"]).flip(0)
    delta = torch.where(inside, delta, 0.0)
    dh0 = torch.where(some[:, None], (f * delta)[first.clamp(max=rows - 1)], s["grad_last"])
    if s["case"]["gate"] == "decay":
        return delta * above, delta, dh0
    g = s["g"].to(f.dtype)
    other = torch.sigmoid(-g)
    return delta * (above - x) * f * other, delta * other, dh0


def _run_plain(s):
    op, t = s["case"]["op"], (s["x"] if "x" in s else s["res"]).dtype
    if op == "embed":
        return {"res": _plain_embed(s)}
    if op == "embed_grad":
        return {"res": _plain_embed_grad(s)}
    if op == "step":
        f, u, _ = _plain_gates(s)
        new = f * s["state"] + u
        return {"h": new.to(t), "new_state": new}
    if op.startswith("norm"):
        v, rstd, y = _plain_norm(s)
        out = {"rstd": rstd}
        if s["residual"] is not None:
            out["sum"] = v.to(t)
        if op == "norm_q8":
            out["res"], out["scales"] = _plain_q8(y, s["case"]["group"])
            return out
        out["res"] = y.to(t)
        if op == "norm_train":
            out["dx"], out["dweight"] = _plain_norm_grad(s, v, rstd)
        return out
    f, x, h, last, starts, into, inside = _plain_scan_forward(s)
    out = {"h": h.to(t), "last": last}
    if op == "scan_train":
        dg, dx, out["dh0"] = _plain_scan_grad(s, f, x, h, starts, into, inside)
        out["dg"], out["dx"] = dg.to(t), dx.to(t)
    return out


# ---- the framework's calls ----

_CODES = {torch.float64: "F64", torch.float32: "F32", torch.float16: "F16", torch.bfloat16: "BF16"}


def _code(t):
    from daphne_b200 import lib
    return getattr(lib, _CODES[t])


def _scratch(s):
    """The working memory that a program keeps for its calls."""
    from daphne_b200.lib import lib
    c = s["case"]
    t, n = _code(TYPES[c["type"]]), 0
    if c["op"] == "embed_grad":
        n = lib.db2k_embed_grad_scratch_bytes(t, c["vocab"], c["cols"], c["rows"])
    elif c["op"] == "norm_train":
        n = lib.db2k_rms_norm_grad_scratch_bytes(t, c["rows"], c["cols"])
    elif c["op"].startswith("scan"):
        n = lib.db2k_gated_scan_scratch_bytes(t, c["rows"], c["cols"], c["seqs"])
    return torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")


def _p(x):
    """Address and leading dimension."""
    return (None, 0) if x is None else (x.data_ptr(), x.shape[1])


def _run_own(s):
    from daphne_b200 import lib as names
    from daphne_b200.lib import check, lib
    c = s["case"]
    op, rows, cols = c["op"], c["rows"], c["cols"]
    t = _code(TYPES[c["type"]])
    stream = torch.cuda.current_stream().cuda_stream
    scratch = (s["scratch"].data_ptr(), s["scratch"].numel())
    if op == "embed":
        check(lib.db2k_embed(t, s["table"].data_ptr(), c["vocab"], cols, cols, names.I64, s["tokens"].data_ptr(), 1, rows,
                             s["scale"], *_p(s["res"]), None, stream))
        return {"res": s["res"]}
    if op == "embed_grad":
        check(lib.db2k_embed_grad(t, *_p(s["grad"]), rows, cols, names.I64, s["tokens"].data_ptr(), 1, s["scale"], t,
                                  s["res"].data_ptr(), c["vocab"], cols, 0, *scratch, None, stream))
        return {"res": s["res"]}
    if op.startswith("norm"):
        front = (t, s["x"].data_ptr(), rows, cols, cols, *_p(s["residual"]), s["weight"].data_ptr(), EPS, *_p(s["sum"]))
        out = {"rstd": s["rstd"], "res": s["res"]}
        if s["residual"] is not None:
            out["sum"] = s["sum"]
        if op == "norm_q8":
            check(lib.db2k_rms_norm_q8(*front, *_p(s["res"]), *_p(s["scales"]), c["group"], s["rstd"].data_ptr(), stream))
            return {**out, "scales": s["scales"]}
        check(lib.db2k_rms_norm(*front, *_p(s["res"]), s["rstd"].data_ptr(), stream))
        if op == "norm_train":
            v = s["sum"] if s["residual"] is not None else s["x"]
            check(lib.db2k_rms_norm_grad(t, *_p(s["grad"]), rows, cols, *_p(v), s["weight"].data_ptr(), s["rstd"].data_ptr(),
                                         *_p(s["dsum"]), *_p(s["dx"]), s["dweight"].data_ptr(), *scratch, stream))
            out["dx"], out["dweight"] = s["dx"], s["dweight"]
        return out
    gate = names.GATE_SIGMOID if c["gate"] == "sigmoid" else names.GATE_DECAY
    if op == "step":
        check(lib.db2k_gated_step(t, gate, *_p(s["g"]), *_p(s["x"]), rows, cols, *_p(s["state"]), *_p(s["new_state"]),
                                  *_p(s["h"]), stream))
        return {"h": s["h"], "new_state": s["new_state"]}
    off = None if s["offsets"] is None else s["offsets"].data_ptr()
    check(lib.db2k_gated_scan(t, gate, *_p(s["g"]), *_p(s["x"]), rows, cols, off, c["seqs"], *_p(s["h0"]), *_p(s["h"]),
                              *_p(s["last"]), *scratch, stream))
    out = {"h": s["h"], "last": s["last"]}
    if op == "scan_train":
        check(lib.db2k_gated_scan_grad(t, gate, *_p(s["g"]), *_p(s["x"]), *_p(s["h"]), *_p(s["grad"]), rows, cols, off,
                                       c["seqs"], *_p(s["h0"]), *_p(s["grad_last"]), *_p(s["dg"]), *_p(s["dx"]),
                                       *_p(s["dh0"]), *scratch, stream))
        out["dg"], out["dx"], out["dh0"] = s["dg"], s["dx"], s["dh0"]
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- from the definitions, in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    op, t = case["op"], TYPES[case["type"]]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point() and v.dtype != torch.float8_e4m3fn}
    if op == "embed":
        res = torch.zeros(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        use = s["tokens"] >= 0
        res[use] = d["table"][s["tokens"][use]] * s["scale"]
        return {"res": res}
    if op == "embed_grad":
        # tokens in order, differences of running sums would cancel: row blocks of one-hot products instead
        tok, use = s["tokens"], s["tokens"] >= 0
        seen, inverse = torch.unique(tok[use], return_inverse=True)
        res = torch.zeros(case["vocab"], case["cols"], dtype=torch.float64, device="cuda")
        rows = d["grad"][use]
        for k in range(0, len(seen), 1024):
            hot = (inverse[None, :] == torch.arange(k, min(k + 1024, len(seen)), device="cuda")[:, None]).double()
            res[seen[k:k + 1024]] = hot @ rows * s["scale"]
        return {"res": res}
    if op.startswith("norm"):
        v = d["x"] if s["residual"] is None else (d["x"] + d["residual"]).to(t).double()
        ms = torch.einsum("rc,rc->r", v, v)[:, None] / case["cols"]
        rstd = 1.0 / torch.sqrt(ms + EPS)
        y = v * d["weight"] * rstd
        out = {"rstd": rstd}
        if s["residual"] is not None:
            out["sum"] = v
        if op == "norm_q8":
            group = case["group"] or case["cols"]
            parts, scales = [], []
            for k in range(0, case["cols"], group):
                part = y[:, k:k + group]
                most = part.abs().max(1, keepdim=True).values
                scale = torch.where(most == 0, 1.0, most / E4M3_MAX)
                parts.append((part / scale).to(torch.float8_e4m3fn).double())
                scales.append(scale)
            out["res"], out["scales"] = torch.cat(parts, 1), torch.cat(scales, 1)
            return out
        out["res"] = y
        if op == "norm_train":
            n = v * rstd  # normalised rows: dx = rstd (t - n <t, n> / C)
            tw = d["grad"] * d["weight"]
            dx = (tw - n * (torch.einsum("rc,rc->r", tw, n)[:, None] / case["cols"])) * rstd
            out["dx"] = dx if s["dsum"] is None else dx + d["dsum"]
            out["dweight"] = torch.einsum("rc,rc->c", d["grad"], n)[None, :]
        return out
    f = d["g"] if case["gate"] == "decay" else 1.0 / (1.0 + torch.exp(-d["g"]))
    u = d["x"] if case["gate"] == "decay" else (1.0 - f) * d["x"]
    if op == "step":
        new = f * d["state"] + u
        return {"h": new, "new_state": new}
    rows = case["rows"]
    lengths = torch.tensor(_lengths(case, seed), device="cuda")
    first = torch.cumsum(lengths, 0) - lengths
    zero = torch.zeros(1, case["cols"], dtype=torch.float64, device="cuda")
    f, u = torch.cat([f, zero + 1.0]), torch.cat([u, zero])  # one row more, which leaves a state as it is
    above = torch.zeros(rows + 1, case["cols"], dtype=torch.float64, device="cuda")
    h, state = torch.zeros_like(above), d["h0"].clone()
    steps = torch.arange(s["longest"], device="cuda")
    at = torch.where(steps[:, None] < lengths[None, :], first[None, :] + steps[:, None], rows)
    for i in at.unbind(0):
        above[i] = state
        state = torch.addcmul(u[i], f[i], state)
        h[i] = state
    h[rows] = 0.0
    out = {"h": h[:rows], "last": state}
    if op == "scan_train":
        grad = torch.cat([d["grad"], zero])
        delta, c = torch.zeros_like(above), d["grad_last"].clone()
        for i in at.flip(0).unbind(0):
            step = c + grad[i]
            delta[i] = step
            c = f[i] * step
        delta = delta[:rows]
        ff, ab = f[:rows], above[:rows]
        if case["gate"] == "decay":
            out["dg"], out["dx"] = delta * ab, delta
        else:
            out["dg"], out["dx"] = delta * (ab - d["x"]) * ff * (1.0 - ff), delta * (1.0 - ff)
        out["dh0"] = c
    return out
