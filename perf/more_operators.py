"""Performance cases of what a recurrent block of a language model needs beside
its filters: the gated linear recurrence (ferrum_gpu.ssm), the root-mean-square
norm of a residual stream (ferrum_gpu.norm) and dropout (ferrum_gpu.pointwise).

A case is a dict of plain values:
  op        "rec"          recurrence of whole sequences, states in and out
            "rec_train"    its forward and backward pass
            "rec_step"     one token per row, state in a cache of slots
            "norm"         residual addition and norm, of the rows' type
            "norm8"        the same, normed rows in 8 bits (e4m3) with scales
            "norm_train"   dropout, residual addition and norm, forward and backward
            "dropout"      elements dropped and scaled, masks from a counter
  dtype     of the rows: "float32", "bfloat16" or "float16"; parameters, states
            and scales are float32
  rec*      batch (sequences, rows of a step), length (tokens of a sequence, the
            longest one's where packed), tokens (0: dense; else of all packed
            sequences, ragged, one of them empty), channels
  norm*     rows, width, group (norm8: elements that share a scale, 0: a row)
  dropout   n elements
  p         dropout's probability

``own`` chooses between the plain form (elementary torch operations in 32 bits,
rounded once at the end) and the calls of the package.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
RATE = 8.0
EPS = 1e-6
E4M3_MOST = 448.0


def _rec(name, op, batch, length, channels, dtype, tokens=0):
    return {"name": name, "op": op, "batch": batch, "length": length, "tokens": tokens, "channels": channels,
            "dtype": dtype}


def _norm(name, op, rows, width, dtype, group=0, p=0.0):
    return {"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype, "group": group, "p": p}


def listed():
    return [
        # A long prompt on its own: few rows, so the time axis has to be split.
        _rec("rec_1x8192x2048_bf16", "rec", 1, 8192, 2048, "bfloat16"),
        # Prompts of different lengths in one call, odd channel count.
        _rec("rec_packed_9_f16", "rec", 9, 2048, 1500, "float16", tokens=7001),
        # The largest: a batch of long prompts through a wide layer.
        _rec("rec_4x2048x4096_bf16", "rec", 4, 2048, 4096, "bfloat16"),
        # An ordinary training step's recurrence, forward and backward.
        _rec("rec_train_4x1024x2048_bf16", "rec_train", 4, 1024, 2048, "bfloat16"),
        # Training on one long sequence in full precision, an odd number of tokens.
        _rec("rec_train_1x4099x1024_f32", "rec_train", 1, 4099, 1024, "float32"),
        # One token of one sequence: latency.
        _rec("rec_step_1x2048_bf16", "rec_step", 1, 1, 2048, "bfloat16"),
        # One token of each sequence of a full serving batch.
        _rec("rec_step_256x4096_bf16", "rec_step", 256, 1, 4096, "bfloat16"),
        # One token's residual stream: latency.
        _norm("norm_1x2048_bf16", "norm", 1, 2048, "bfloat16"),
        # Prompts into a product that takes 8 bits with a scale for 128 elements.
        _norm("norm8_8192x4096_bf16", "norm8", 8192, 4096, "bfloat16", group=128),
        # A training step's residual stream with dropout, forward and backward.
        _norm("norm_train_8192x4096_bf16", "norm_train", 8192, 4096, "bfloat16", p=0.1),
        # Odd sizes, one scale for a row.
        _norm("norm8_2003x1500_f16", "norm8", 2003, 1500, "float16"),
        # A training step's activations.
        {"name": "dropout_32m_bf16", "op": "dropout", "n": 8 * 1024 * 4096, "dtype": "bfloat16", "p": 0.1},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: every operator and type, lengths and rows from one to
    many, odd and ragged sizes, at most the largest listed case's work."""
    op = rng.choice(["rec", "rec", "rec_train", "rec_train", "rec_step", "norm", "norm8", "norm_train", "dropout"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "dropout":
        return {"op": op, "n": _spread(rng, 1000, 1 << 25), "dtype": dtype, "p": rng.choice([0.05, 0.1, 0.5])}
    channels = _spread(rng, 128, 4096)
    if rng.random() < 0.6:
        channels = max(64, channels // 64 * 64)
    if op.startswith("norm"):
        rows = _spread(rng, 1, min(16384, (1 << 24) // channels))
        return {"op": op, "rows": rows, "width": channels, "dtype": dtype,
                "group": rng.choice([0, 128]) if op == "norm8" else 0,
                "p": rng.choice([0.0, 0.1]) if op == "norm_train" else 0.0}
    if op == "rec_step":
        return {"op": op, "batch": _spread(rng, 1, 512), "length": 1, "tokens": 0, "channels": channels,
                "dtype": dtype}
    pairs = ((1 << 24) if op == "rec" else (1 << 23)) // channels
    length = _spread(rng, 1, min(8192, pairs))
    batch = max(1, min(64, _spread(rng, 1, max(1, pairs // length))))
    tokens = 0
    if batch >= 3 and rng.random() < 0.35:
        # ragged: a third to most of what a dense call would hold
        tokens = min(max(1, int(batch * length * rng.uniform(0.3, 0.8))), (batch - 1) * length)
    return {"op": op, "batch": batch, "length": length, "tokens": tokens, "channels": channels, "dtype": dtype}


# ---------------------------------------------------------------- inputs


def _lengths(case, g):
    """Lengths of the packed sequences: one empty, none above `length`."""
    n, most, left = case["batch"], case["length"], case["tokens"]
    share = torch.rand(n - 1, generator=g).add_(0.05)
    got = (share / share.sum() * left).floor().clamp_(max=most).long()
    room = most - got
    before = torch.cumsum(room, 0) - room
    got += torch.minimum(room, (left - got.sum() - before).clamp_(min=0))
    return torch.cat([got[:1], torch.zeros(1, dtype=torch.long), got[1:]])


def _inputs(case, seed):
    """The tensors that a program has before the call, from the seed alone."""
    host = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    t, op, s = TYPES[case["dtype"]], case["op"], {}
    # a program's running count of random numbers
    s["seed"], s["offset"] = 1234 + seed, 1000 * (seed % 97)
    if op == "dropout":
        s["x"] = normal(case["n"]).to(t)
        return s
    if op.startswith("norm"):
        n, d = case["rows"], case["width"]
        s["x"], s["residual"] = normal(n, d).to(t), (3 * normal(n, d)).to(t)
        s["weight"] = 1 + 0.2 * normal(d)
        if op == "norm_train":
            s["grad"], s["grad_sum"] = normal(n, d).to(t), normal(n, d).to(t)
        return s
    d, b = case["channels"], case["batch"]
    step = op == "rec_step"
    rows = (b,) if step or case["tokens"] else (b, case["length"])
    if case["tokens"]:
        rows = (case["tokens"],)
        ends = torch.cumsum(_lengths(case, host), 0)
        s["offsets"] = torch.cat([ends.new_zeros(1), ends]).to(torch.int32).cuda()
    if step:
        s["slots"] = torch.randperm(b, generator=host).to(torch.int32).cuda()
    # one projection's halves: what is filtered, and the other branch; the gates' projection
    s["x"] = normal(*rows, 2 * d).to(t)[..., :d]
    gates = normal(*rows, 2 * d).to(t)
    s["gate_a"], s["gate_x"] = gates[..., :d], gates[..., d:]
    s["bias_a"], s["bias_x"] = 0.5 * normal(d), 0.5 * normal(d)
    # a full gate keeps between 0.9 and 0.999 of the state
    kept = -torch.log(0.9 + 0.099 * uniform(d)) / RATE
    s["decay"] = torch.log(torch.expm1(kept))
    s["state"] = normal(b, d)
    if op == "rec_train":
        s["grad"] = normal(*rows, d).to(t)
    return s


def prepare(case, seed):
    """Inputs, room for the outputs, and the plan that a program keeps."""
    s = _inputs(case, seed)
    s["case"] = case
    op = case["op"]
    s["out"] = torch.empty(s["x"].shape, dtype=s["x"].dtype, device="cuda")
    if op.startswith("norm"):
        n, d, group = case["rows"], case["width"], case["group"]
        s["sum"] = torch.empty_like(s["x"])
        if op == "norm8":
            s["out"] = torch.empty((n, d), dtype=torch.float8_e4m3fn, device="cuda")
            s["scales"] = torch.empty((n, -(-d // group) if group else 1), device="cuda")
        if op == "norm_train":
            s["grads"] = {"x": torch.empty_like(s["x"]), "residual": torch.empty_like(s["x"]),
                          "weight": torch.empty_like(s["weight"])}
        if own:
            s["plan"] = _package().norm.NormPlan(n, d, _dev(), dtype=case["dtype"], eps=EPS, group=group)
    elif op.startswith("rec"):
        if op == "rec_train":
            s["grads"] = {k: torch.empty(s[k].shape, dtype=s[k].dtype, device="cuda")
                          for k in ("x", "gate_a", "gate_x", "decay", "bias_a", "bias_x")}
        else:
            s["state_out"] = torch.empty_like(s["state"])
        if own and op != "rec_step":
            s["plan"] = _package().ssm.RecurrencePlan(case["batch"], case["length"], case["channels"], _dev(),
                                                      dtype=case["dtype"], rate=RATE, tokens=case["tokens"] or None)
            if op == "rec_train":
                s["checkpoints"] = torch.empty(s["plan"].checkpoint_bytes, dtype=torch.uint8, device="cuda")
    if own:
        _dev()
    torch.cuda.synchronize()  # the package's stream is not torch's
    return s


_device = None


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrum-gpu_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ferrum_gpu

    return ferrum_gpu


def _dev():
    global _device
    if _device is None:
        _device = _package().hip.Device(0)
    return _device


# ---------------------------------------------------------------- one pass


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    case = s["case"]
    op = case["op"]
    if op == "dropout":
        _package().pointwise.dropout(_dev(), s["x"], s["out"], case["n"], case["p"], s["seed"], offset=s["offset"])
        return s["out"]
    if op == "norm":
        s["plan"].forward(s["x"], s["out"], weight=s["weight"], residual=s["residual"], sum_out=s["sum"])
        return [s["out"], s["sum"]]
    if op == "norm8":
        s["plan"].forward(s["x"], s["out"], weight=s["weight"], residual=s["residual"], sum_out=s["sum"],
                          scales=s["scales"])
        return [s["out"], s["scales"], s["sum"]]
    if op == "norm_train":
        g, drop = s["grads"], {"dropout": case["p"], "seed": s["seed"], "offset": s["offset"]}
        s["plan"].forward(s["x"], s["out"], weight=s["weight"], residual=s["residual"], sum_out=s["sum"], **drop)
        s["plan"].backward(s["sum"], s["grad"], weight=s["weight"], grad_sum=s["grad_sum"], grad_x=g["x"],
                           grad_residual=g["residual"], grad_weight=g["weight"], **drop)
        return {"out": s["out"], "sum": s["sum"], **g}
    args = (s["x"], s["gate_a"], s["gate_x"], s["decay"])
    bias = {"bias_a": s["bias_a"], "bias_x": s["bias_x"]}
    if op == "rec_step":
        _package().ssm.recurrence_step(_dev(), *args, s["state"], s["out"], slots=s["slots"],
                                       state_out=s["state_out"], rate=RATE, **bias)
        return [s["out"], s["state_out"]]
    offsets = s.get("offsets")
    if op == "rec":
        s["plan"].forward(*args, s["out"], initial=s["state"], final=s["state_out"], offsets=offsets, **bias)
        return [s["out"], s["state_out"]]
    g = s["grads"]
    s["plan"].forward(*args, s["out"], offsets=offsets, checkpoints=s["checkpoints"], **bias)
    s["plan"].backward(*args, s["grad"], s["checkpoints"], offsets=offsets, **bias,
                       **{"grad_" + k: v for k, v in g.items()})
    return {"out": s["out"], **g}


# The plain forms: elementary torch operations in 32 bits.


def _f(x):
    return x.to(torch.float32)


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _running(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, from h = 0, in log2(tokens)
    doublings of the span that each h_t covers."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _rec_terms(s):
    """x, both gates, the full gate's logarithm of the kept share, the share and the input's factor."""
    x = _f(s["x"])
    x = x if x.dim() == 3 else x[None]
    r = torch.sigmoid(_f(s["gate_a"]).reshape(x.shape) + s["bias_a"])
    i = torch.sigmoid(_f(s["gate_x"]).reshape(x.shape) + s["bias_x"])
    full = -RATE * _softplus(s["decay"])
    log_a = full * r
    return x, r, i, full, torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a))


def _starts(s):
    """Packed sequences: which of them have tokens, and their first and last."""
    at = s["offsets"].long()
    some = torch.nonzero(at[1:] > at[:-1])[:, 0]
    return some, at[:-1][some], at[1:][some] - 1


def _plain_rec(s):
    x, _, i, _, a, m = _rec_terms(s)
    b = m * i * x
    final = s["state"].clone()
    if "offsets" in s:
        some, first, last = _starts(s)
        b[0, first] += a[0, first] * s["state"][some]
        a[0, first] = 0
        h = _running(a, b)
        final[some] = h[0, last]
    else:
        b[:, 0] += a[:, 0] * s["state"]
        h = _running(a, b)
        final = h[:, -1].clone()
    return [h.reshape(s["out"].shape).to(s["out"].dtype), final]


def _plain_rec_train(s):
    x, r, i, full, a, m = _rec_terms(s)
    held = a
    if "offsets" in s:
        _, first, _ = _starts(s)
        held = a.clone()
        held[0, first] = 0
    h = _running(held, m * i * x)
    # the reverse run: g_t = grad_t + a_{t+1} g_{t+1}
    after = torch.cat([held[:, 1:], torch.zeros_like(held[:, :1])], 1)
    g = _running(after.flip(1), _f(s["grad"]).reshape(x.shape).flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    d_log = g * (held * before - i * x * a * a / m)
    d_a = d_log * full * r * (1 - r)
    d_x = g * m * x * i * (1 - i)

    def like(y):
        return y.reshape(s["out"].shape).to(s["out"].dtype)

    return {"out": like(h), "x": like(g * m * i), "gate_a": like(d_a), "gate_x": like(d_x),
            "decay": (d_log * r).sum((0, 1)) * -RATE * torch.sigmoid(s["decay"]), "bias_a": d_a.sum((0, 1)),
            "bias_x": d_x.sum((0, 1))}


def _plain_rec_step(s):
    x, _, i, _, a, m = _rec_terms(s)
    slots = s["slots"].long()
    h = a[0] * s["state"][slots] + (m * i * x)[0]
    new = s["state"].clone()
    new[slots] = h
    return [h.to(s["out"].dtype), new]


_GOLDEN, _MIX1, _MIX2 = (v - (1 << 64) for v in (0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB))


def _shift(z, k):
    """z >> k of 64 bits without a sign."""
    return (z >> k) & ((1 << (64 - k)) - 1)


def _kept(s, n):
    """Which of n elements dropout keeps: element i takes half i % 2 of the
    seed's splitmix64 number offset + i / 2."""
    z = torch.arange((n + 1) // 2, device="cuda", dtype=torch.int64) + (s["offset"] + 1)
    z = z * _GOLDEN + s["seed"]
    z = (z ^ _shift(z, 30)) * _MIX1
    z = (z ^ _shift(z, 27)) * _MIX2
    z = z ^ _shift(z, 31)
    bits = torch.stack([z & 0xFFFFFFFF, _shift(z, 32)], -1).reshape(-1)[:n]
    return bits >= round(s["case"]["p"] * (1 << 32))


def _dropped(x, s):
    p = s["case"]["p"]
    return torch.where(_kept(s, x.numel()).reshape(x.shape), x * (1 / (1 - p)), 0) if p else x


def _plain_dropout(s):
    return _dropped(_f(s["x"]), s).to(s["x"].dtype)


def _plain_norm(s):
    v = _dropped(_f(s["x"]), s) + _f(s["residual"])
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * s["weight"]
    t = s["x"].dtype
    if s["case"]["op"] == "norm":
        return [y.to(t), v.to(t)]
    if s["case"]["op"] == "norm8":
        n, d = y.shape
        group = s["case"]["group"] or d
        parts = torch.nn.functional.pad(y, (0, -d % group)).reshape(n, -1, group)
        scales = parts.abs().amax(-1) / E4M3_MOST
        q = parts / torch.where(scales > 0, scales, 1)[..., None]
        return [q.reshape(n, -1)[:, :d].to(torch.float8_e4m3fn), scales, v.to(t)]
    # the backward pass: of the sum as it was stored
    total = v.to(t)
    u, dy = _f(total), _f(s["grad"])
    rstd = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
    dn = dy * s["weight"]
    dv = rstd * (dn - u * rstd * rstd * (dn * u).mean(-1, keepdim=True)) + _f(s["grad_sum"])
    return {"out": y.to(t), "sum": total, "x": _dropped(dv, s).to(t), "residual": dv.to(t),
            "weight": (dy * u * rstd).sum(0)}


_PLAIN = {"rec": _plain_rec, "rec_train": _plain_rec_train, "rec_step": _plain_rec_step, "norm": _plain_norm,
          "norm8": _plain_norm, "norm_train": _plain_norm, "dropout": _plain_dropout}


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    """The definitions in 64 bits: the recurrence token after token, dense
    sequences side by side, packed ones one after another."""
    s = _inputs(case, seed)
    if case["op"].startswith("rec"):
        s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
        return _exact_rec(case, s)
    if case["op"] == "dropout":
        return _exact_drop(case, s, s["x"].double())
    return _exact_norm(case, s)


def _exact_bits(seed, offset, n):
    """The seed's splitmix64 numbers, offset and on, as 32-bit halves."""
    with np.errstate(over="ignore"):
        z = (np.arange(offset + 1, offset + 1 + (n + 1) // 2, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
             + np.uint64(seed))
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    z ^= z >> np.uint64(31)
    return torch.from_numpy(z.view(np.uint32).astype(np.int64)[:n]).cuda()


def _exact_drop(case, s, x):
    if case["p"] == 0:
        return x
    keep = _exact_bits(s["seed"], s["offset"], x.numel()).reshape(x.shape) >= round(case["p"] * 2 ** 32)
    return x * keep / (1 - case["p"])


def _exact_norm(case, s):
    v = _exact_drop(case, s, s["x"].double()) + s["residual"].double()
    w = s["weight"].double()
    y = v / torch.sqrt((v ** 2).sum(-1, keepdim=True) / case["width"] + EPS) * w
    if case["op"] == "norm":
        return [y, v]
    if case["op"] == "norm8":
        group = case["group"] or case["width"]
        scales = torch.stack([p.abs().max(-1).values for p in y.split(group, -1)], -1) / E4M3_MOST
        q = torch.cat([p / scales[:, k:k + 1] for k, p in enumerate(y.split(group, -1))], -1)
        return [q, scales, v]
    # the stored sum is what the backward pass is given
    u = _stored_sum(case, s).double()
    norm = torch.sqrt((u ** 2).sum(-1, keepdim=True) / case["width"] + EPS)
    g = s["grad"].double()
    along = (g * w * u).sum(-1, keepdim=True) / case["width"]
    dv = g * w / norm - u * along / norm ** 3 + s["grad_sum"].double()
    return {"out": y, "sum": v, "x": _exact_drop(case, s, dv), "residual": dv, "weight": (g * u / norm).sum(0)}


def _stored_sum(case, s):
    """The sum that the forward pass stores, added in 32 bits and rounded to the rows' type."""
    p, x = case["p"], s["x"].float()
    if p:
        keep = _exact_bits(s["seed"], s["offset"], x.numel()).reshape(x.shape) >= round(p * 2 ** 32)
        x = torch.where(keep, x * (1 / (1 - p)), torch.zeros_like(x))
    return (x + s["residual"].float()).to(s["residual"].dtype)


def _exact_rec(case, s):
    r = 1 / (1 + torch.exp(-(s["gate_a"] + s["bias_a"])))
    i = 1 / (1 + torch.exp(-(s["gate_x"] + s["bias_x"])))
    full = -RATE * torch.log1p(torch.exp(s["decay"]))
    log_a = full * r
    a, m = torch.exp(log_a), torch.sqrt(1 - torch.exp(2 * log_a))
    x = s["x"]
    if case["op"] == "rec_step":
        slots, new = s["slots"].long(), s["state"].clone()
        new[slots] = a * s["state"][slots] + m * i * x
        return [new[slots], new]
    train = case["op"] == "rec_train"
    if case["tokens"]:
        ends = s["offsets"].tolist()
        spans = [(slice(ends[k], ends[k + 1]), k) for k in range(case["batch"]) if ends[k + 1] > ends[k]]
    else:
        spans = [(slice(None), None)]
    out, final, g_all = torch.zeros_like(x), s["state"].clone(), torch.zeros_like(x)
    before = torch.zeros_like(x)
    for at, k in spans:
        dense = k is None
        aa, bb = ((a, m * i * x) if dense else (a[at][None], (m * i * x)[at][None]))
        h = torch.zeros_like(aa[:, 0]) if train else s["state"] if dense else s["state"][k][None]
        ys, hs = [], []
        for t in range(aa.shape[1]):
            hs.append(h)
            h = aa[:, t] * h + bb[:, t]
            ys.append(h)
        y, b4 = torch.stack(ys, 1), torch.stack(hs, 1)
        if dense:
            out, final, before = y, h, b4
        else:
            out[at], final[k], before[at] = y[0], h[0], b4[0]
        if train:
            gr = s["grad"] if dense else s["grad"][at][None]
            carry, gs = torch.zeros_like(h), []
            for t in range(aa.shape[1] - 1, -1, -1):
                g = gr[:, t] + carry
                gs.append(g)
                carry = g * aa[:, t]
            g = torch.stack(gs[::-1], 1)
            if dense:
                g_all = g
            else:
                g_all[at] = g[0]
    if not train:
        return [out, final]
    axes = tuple(range(x.dim() - 1))
    d_a = g_all * (before - i * x * a / m)
    d_log = d_a * a
    d_ga = d_log * full * r * (1 - r)
    d_gx = g_all * m * x * i * (1 - i)
    return {"out": out, "x": g_all * m * i, "gate_a": d_ga, "gate_x": d_gx,
            "decay": (d_log * r).sum(axes) * -RATE / (1 + torch.exp(-s["decay"])), "bias_a": d_ga.sum(axes),
            "bias_x": d_gx.sum(axes)}


# ---------------------------------------------------------------- the work


def work(case):
    """Each input read and each output written once; the operations of the
    formulas, an exponential, reciprocal or root as one: for the recurrence 2 x
    4 for the gates, 8 for the share and the factor, 4 for the state, 24 more
    for the gradients; for the norm 6, 16 more for its gradients; for dropout 4
    (8 where it stands before a norm, both ways)."""
    op, e = case["op"], BYTES[case["dtype"]]
    if op == "dropout":
        return {"bytes": 2 * e * case["n"], "flops": 4 * case["n"]}
    if op.startswith("norm"):
        n, d = case["rows"], case["width"]
        if op == "norm_train":
            return {"bytes": 8 * e * n * d + 8 * d, "flops": (30 if case["p"] else 22) * n * d}
        if op == "norm8":
            scales = n * (-(-d // case["group"]) if case["group"] else 1)
            return {"bytes": (3 * e + 1) * n * d + 4 * d + 4 * scales, "flops": 8 * n * d}
        return {"bytes": 4 * e * n * d + 4 * d, "flops": 6 * n * d}
    d, b = case["channels"], case["batch"]
    rows = b if op == "rec_step" else case["tokens"] or b * case["length"]
    if op == "rec_train":
        # x, both gates, the output's gradient; the output and three gradients
        return {"bytes": 8 * e * rows * d + 24 * d, "flops": 44 * rows * d}
    return {"bytes": 4 * e * rows * d + 12 * d + 8 * b * d, "flops": 20 * rows * d}
