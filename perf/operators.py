"""Performance cases of the sequence filters (ferrum_gpu.ssm): the short causal
convolution and the selective state space scan, over whole sequences (prompts,
training) and for single tokens.

A case is a dict of plain values:
  op        "conv"        causal convolution of sequences, states in and out
            "conv_train"  its forward and backward pass
            "conv_step"   one token per row, window state in a cache of slots
            "scan"        selective scan of sequences, states in and out
            "scan_train"  its forward and backward pass
            "scan_step"   one token per row, state in a cache of slots
  batch     sequences (rows of a step)
  length    tokens of a sequence; the longest one's where packed
  tokens    0: every sequence has `length` tokens; else the tokens of all
            sequences, packed one after another, ragged, one of them empty
  channels, width (conv), states and groups (scan)
  dtype     of the rows: "float32", "bfloat16" or "float16"; parameters and
            scan states are float32

``own`` chooses between the plain form (elementary torch operations in 32 bits,
rounded once at the end) and the calls of ferrum_gpu.ssm.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def _case(name, op, batch, length, channels, dtype, width=0, states=0, groups=0, tokens=0):
    return {"name": name, "op": op, "batch": batch, "length": length, "tokens": tokens, "channels": channels,
            "width": width, "states": states, "groups": groups, "dtype": dtype}


def listed():
    return [
        # A prompt of a mid-sized layer, an odd number of tokens.
        _case("conv_2x1001x2048_bf16", "conv", 2, 1001, 2048, "bfloat16", width=4),
        # Prompts of different lengths in one call, odd channel count.
        _case("conv_packed_9_f16", "conv", 9, 2048, 1500, "float16", width=3, tokens=7001),
        # A training step's convolution, forward and backward.
        _case("conv_train_8x2048x4096_bf16", "conv_train", 8, 2048, 4096, "bfloat16", width=4),
        # One token of one sequence: latency.
        _case("conv_step_1x2048_f32", "conv_step", 1, 1, 2048, "float32", width=4),
        # One token of each sequence of a full serving batch.
        _case("conv_step_256x4096_bf16", "conv_step", 256, 1, 4096, "bfloat16", width=4),
        # A short prompt on its own: few rows, so the time axis has to be split.
        _case("scan_1x512x2048_bf16", "scan", 1, 512, 2048, "bfloat16", states=16, groups=1),
        # Prompts of different lengths in one call, two groups, few states.
        _case("scan_packed_7_f16", "scan", 7, 4096, 1536, "float16", states=8, groups=2, tokens=9001),
        # The largest: a batch of long prompts through a wide layer.
        _case("scan_4x2048x4096_bf16", "scan", 4, 2048, 4096, "bfloat16", states=16, groups=1),
        # Training on one long sequence in full precision.
        _case("scan_train_1x4099x1024_f32", "scan_train", 1, 4099, 1024, "float32", states=16, groups=1),
        # An ordinary training step's scan, forward and backward.
        _case("scan_train_4x1024x2048_bf16", "scan_train", 4, 1024, 2048, "bfloat16", states=16, groups=1),
        # One token of one sequence: latency.
        _case("scan_step_1x2048_bf16", "scan_step", 1, 1, 2048, "bfloat16", states=16, groups=1),
        # One token of each sequence of a full serving batch.
        _case("scan_step_256x4096_bf16", "scan_step", 256, 1, 4096, "bfloat16", states=16, groups=1),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: every operator and type, lengths from one token to long
    ones, odd and ragged sizes, at most the largest listed case's work."""
    op = rng.choice(["conv", "conv_train", "conv_step", "scan", "scan", "scan_train", "scan_train", "scan_step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    channels = _spread(rng, 256, 4096)
    if rng.random() < 0.6:
        channels = max(64, channels // 64 * 64)
    width = states = groups = 0
    if op.startswith("conv"):
        width = rng.choice([2, 3, 4, 4, 4, 5, 8])
    else:
        states = rng.choice([4, 8, 13, 16, 16, 16, 16, 24, 32, 64])
        groups = rng.choice([1, 1, 1, 2, 4])
        channels = max(groups, channels // groups * groups)
    if op.endswith("step"):
        batch = _spread(rng, 1, 512)
        return {"op": op, "batch": batch, "length": 1, "tokens": 0, "channels": channels, "width": width,
                "states": states, "groups": groups, "dtype": dtype}
    # (token, channel) pairs times states: at most what the largest case of the kind has
    most = {"conv": 1 << 26, "conv_train": 1 << 25, "scan": 1 << 29, "scan_train": 1 << 27}[op]
    pairs = most // (channels * max(1, (states + 15) // 16 * 16))
    length = _spread(rng, 1, max(1, min(8192, pairs)))
    batch = max(1, min(64, _spread(rng, 1, max(1, pairs // length))))
    tokens = 0
    if batch >= 3 and rng.random() < 0.35:
        # ragged: a third to all of what a dense call would hold
        tokens = max(1, int(batch * length * rng.uniform(0.3, 0.8)))
        tokens = min(tokens, (batch - 1) * length)
    return {"op": op, "batch": batch, "length": length, "tokens": tokens, "channels": channels, "width": width,
            "states": states, "groups": groups, "dtype": dtype}


# ---------------------------------------------------------------- inputs


def _lengths(case, g):
    """Lengths of the packed sequences: one empty, none above `length`."""
    n, most, left = case["batch"], case["length"], case["tokens"]
    share = torch.rand(n - 1, generator=g).add_(0.05)
    got = (share / share.sum() * left).floor().clamp_(max=most).long()
    # what rounding and the cap left over, to the first that have room
    room = most - got
    before = torch.cumsum(room, 0) - room
    got += torch.minimum(room, (left - got.sum() - before).clamp_(min=0))
    return torch.cat([got[:1], torch.zeros(1, dtype=torch.long), got[1:]])


def _rows_shape(case):
    return (case["tokens"],) if case["tokens"] else (case["batch"], case["length"])


def _inputs(case, seed):
    """The tensors that a program has before the call, from the seed alone."""
    host = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    t = TYPES[case["dtype"]]
    d, b = case["channels"], case["batch"]
    step = case["op"].endswith("step")
    rows = (b,) if step else _rows_shape(case)
    s = {}
    if case["tokens"]:
        ends = torch.cumsum(_lengths(case, host), 0)
        s["offsets"] = torch.cat([ends.new_zeros(1), ends]).to(torch.int32).cuda()
    if step:
        s["slots"] = torch.randperm(b, generator=host).to(torch.int32).cuda()
    # the two halves of one projection: what is filtered, and its gate
    both = normal(*rows, 2 * d).to(t)
    if case["op"].startswith("conv"):
        w = case["width"]
        s["x"] = both[..., :d]
        s["weight"] = (uniform(d, w) * 2 - 1) / math.sqrt(w)
        s["bias"] = (uniform(d) * 2 - 1) / math.sqrt(w)
        s["state"] = normal(b, w - 1, d).to(t)
    else:
        n, gr = case["states"], case["groups"]
        s["u"] = torch.nn.functional.silu(normal(*rows, d)).to(t)
        s["z"] = both[..., d:]
        s["delta"] = (0.5 * normal(*rows, d)).to(t)
        # time steps between 0.001 and 0.1 before the token's own part
        rest = torch.exp(uniform(d) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["delta_bias"] = rest + torch.log(-torch.expm1(-rest))
        rank = (d + 15) // 16
        proj = normal(*rows, rank + 2 * gr * n).to(t)
        s["B"] = proj[..., rank:rank + gr * n]
        s["C"] = proj[..., rank + gr * n:]
        s["A"] = -torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * (0.75 + 0.5 * uniform(d, n))
        s["D"] = 0.5 + uniform(d)
        s["state"] = normal(b, d, n)
    if case["op"].endswith("train"):
        s["grad"] = normal(*rows, d).to(t)
    return s


def prepare(case, seed):
    """Inputs, room for the outputs, and the plan that a program keeps."""
    s = _inputs(case, seed)
    s["case"] = case
    op, d = case["op"], case["channels"]
    rows = s["x"] if op.startswith("conv") else s["u"]
    s["out"] = torch.empty(rows.shape, dtype=rows.dtype, device="cuda")
    if op.endswith("train"):
        s["grads"] = {k: torch.empty(s[k].shape, dtype=s[k].dtype, device="cuda")
                      for k in (("x", "weight", "bias") if op == "conv_train"
                                else ("u", "delta", "A", "B", "C", "D", "z", "delta_bias"))}
    else:
        s["state_out"] = torch.empty_like(s["state"])
    if own:
        ssm = _ssm()
        tokens = case["tokens"] or None
        if op in ("conv", "conv_train"):
            s["plan"] = ssm.ConvPlan(case["batch"], case["length"], d, case["width"], _dev(), dtype=case["dtype"],
                                     tokens=tokens)
        if op in ("scan", "scan_train"):
            s["plan"] = ssm.ScanPlan(case["batch"], case["length"], d, case["states"], _dev(),
                                     groups=case["groups"], dtype=case["dtype"], tokens=tokens)
        if op == "scan_train":
            s["checkpoints"] = torch.empty(s["plan"].checkpoint_bytes, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()  # the framework's stream is not torch's
    return s


_device = None


def _ssm():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrum-gpu_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ferrum_gpu

    return ferrum_gpu.ssm


def _dev():
    global _device
    if _device is None:
        _ssm()
        import ferrum_gpu

        _device = ferrum_gpu.hip.Device(0)
    return _device


# ---------------------------------------------------------------- one pass


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    case = s["case"]
    op = case["op"]
    if op == "conv_step":
        _ssm().conv_step(_dev(), s["x"], s["weight"], s["state"], s["out"], bias=s["bias"], slots=s["slots"],
                         state_out=s["state_out"])
        return [s["out"], s["state_out"]]
    if op == "scan_step":
        _ssm().scan_step(_dev(), s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], s["out"], D=s["D"],
                         z=s["z"], delta_bias=s["delta_bias"], slots=s["slots"], state_out=s["state_out"])
        return [s["out"], s["state_out"]]
    offsets = s.get("offsets")
    if op == "conv":
        s["plan"].forward(s["x"], s["weight"], s["out"], bias=s["bias"], initial=s["state"], final=s["state_out"],
                          offsets=offsets)
        return [s["out"], s["state_out"]]
    if op == "scan":
        s["plan"].forward(s["u"], s["delta"], s["A"], s["B"], s["C"], s["out"], D=s["D"], z=s["z"],
                          delta_bias=s["delta_bias"], initial=s["state"], final=s["state_out"], offsets=offsets)
        return [s["out"], s["state_out"]]
    g = s["grads"]
    if op == "conv_train":
        s["plan"].forward(s["x"], s["weight"], s["out"], bias=s["bias"], offsets=offsets)
        s["plan"].backward(s["x"], s["weight"], s["grad"], grad_x=g["x"], grad_weight=g["weight"],
                           grad_bias=g["bias"], bias=s["bias"], offsets=offsets)
    else:
        s["plan"].forward(s["u"], s["delta"], s["A"], s["B"], s["C"], s["out"], D=s["D"], z=s["z"],
                          delta_bias=s["delta_bias"], offsets=offsets, checkpoints=s["checkpoints"])
        s["plan"].backward(s["u"], s["delta"], s["A"], s["B"], s["C"], s["grad"], s["checkpoints"],
                           grad_u=g["u"], grad_delta=g["delta"], grad_A=g["A"], grad_B=g["B"], grad_C=g["C"],
                           D=s["D"], z=s["z"], delta_bias=s["delta_bias"], grad_D=g["D"], grad_z=g["z"],
                           grad_delta_bias=g["delta_bias"], offsets=offsets)
    return {"out": s["out"], **g}


# The plain forms: elementary torch operations in 32 bits.


def _f(x):
    return x.to(torch.float32)


def _marks(s, rows):
    """For each token: its sequence's first token, and one past its last one,
    as places on the time axis (of every batch row alike where dense)."""
    if "offsets" not in s:
        n = rows.shape[1]
        i = torch.zeros(n, dtype=torch.long, device="cuda")
        return i, i + n
    at = s["offsets"].long()
    i = torch.arange(rows.shape[-2], device="cuda")
    of = torch.searchsorted(at[1:].contiguous(), i, right=True)
    return at[of], at[of + 1]


def _conv_window(s):
    """x and what precedes it, [sequences or 1, tokens, channels, width]: the
    rows that each output takes, zeros before a sequence without a state."""
    x = _f(s["x"])
    x = x if x.dim() == 3 else x[None]
    w = s["weight"].shape[1]
    first, _ = _marks(s, x)
    t = torch.arange(x.shape[1], device="cuda")
    src = t[:, None] - (w - 1) + torch.arange(w, device="cuda")  # [tokens, width]
    inside = src >= first[:, None]
    rows = x[:, src.clamp(min=0)] * inside[None, :, :, None]
    if s["case"]["op"] == "conv":
        st = _f(s["state"])
        back = (src - first[:, None] + (w - 1)).clamp(max=max(0, w - 2))  # the state's row, where outside
        if "offsets" in s:
            of = torch.searchsorted(s["offsets"][1:].contiguous(), t.to(torch.int32), right=True)
            prior = st[of[:, None], back][None]
        else:
            prior = st[:, back]
        rows = torch.where(inside[None, :, :, None], rows, prior)
    return rows.transpose(2, 3)


def _like(y, s):
    return y.reshape(s["out"].shape).to(s["out"].dtype)


def _plain_conv(s):
    win = _conv_window(s)
    p = (win * s["weight"]).sum(-1) + s["bias"]
    y = p * torch.sigmoid(p)
    # the last width - 1 rows of (state, sequence)
    x, w = _f(s["x"]), s["weight"].shape[1]
    st = _f(s["state"])
    if "offsets" in s:
        start, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
        x = x.expand(st.shape[0], -1, -1)
    else:
        start = torch.zeros(st.shape[0], dtype=torch.long, device="cuda")
        end = start + x.shape[1]
    k = end[:, None] - (w - 1) + torch.arange(w - 1, device="cuda") - start[:, None]  # place within the sequence
    seq = torch.arange(st.shape[0], device="cuda")[:, None]
    taken = x[seq, (k + start[:, None]).clamp(min=0, max=x.shape[1] - 1)]
    kept = st[seq, (k + (w - 1)).clamp(max=max(0, w - 2))]
    final = torch.where((k >= 0)[:, :, None], taken, kept)
    return [_like(y, s), final.to(s["state"].dtype)]


def _plain_conv_train(s):
    win = _conv_window(s)
    p = (win * s["weight"]).sum(-1) + s["bias"]
    sig = torch.sigmoid(p)
    dp = _f(s["grad"]).reshape(p.shape) * sig * (1 + p * (1 - sig))
    w = s["weight"].shape[1]
    _, last = _marks(s, p)
    t = torch.arange(p.shape[1], device="cuda")
    dst = t[:, None] + (w - 1) - torch.arange(w, device="cuda")  # the output that tap k of this row went to
    inside = dst < last[:, None]
    taken = dp[:, dst.clamp(max=p.shape[1] - 1)] * inside[None, :, :, None]
    dx = (taken.transpose(2, 3) * s["weight"]).sum(-1)
    dw = (win * dp[..., None]).sum((0, 1))
    return {"out": _like(p * sig, s), "x": _like(dx, s), "weight": dw, "bias": dp.sum((0, 1))}


def _plain_conv_step(s):
    slots = s["slots"].long()
    win = torch.cat([_f(s["state"])[slots], _f(s["x"])[:, None]], 1)  # [rows, width, channels]
    p = (win.transpose(1, 2) * s["weight"]).sum(-1) + s["bias"]
    new = s["state"].clone()
    new[slots] = win[:, 1:].to(new.dtype)
    return [_like(p * torch.sigmoid(p), s), new]


def _running(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, from h = 0, in log2(tokens)
    doublings of the span that each h_t covers."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _per_channel(x, s):
    """[.., groups * states] to [sequences or 1, tokens, channels, states], each channel its group's."""
    gr, n, d = s["case"]["groups"], s["case"]["states"], s["case"]["channels"]
    x = _f(x).reshape(-1, *s["u"].shape[-2:-1], gr, 1, n)
    return x.expand(-1, -1, -1, d // gr, -1).reshape(*x.shape[:2], d, n)


def _scan_terms(s):
    u = _f(s["u"])
    u = u if u.dim() == 3 else u[None]
    raw = _f(s["delta"]).reshape(u.shape) + s["delta_bias"]
    dt = _softplus(raw)
    decay = torch.exp(dt[..., None] * s["A"])
    bx = (dt * u)[..., None] * _per_channel(s["B"], s)
    return u, raw, dt, decay, bx


def _starts(s):
    """Packed sequences: which of them have tokens, and their first and last."""
    at = s["offsets"].long()
    some = torch.nonzero(at[1:] > at[:-1])[:, 0]
    return some, at[:-1][some], at[1:][some] - 1


def _plain_scan(s):
    u, _, _, decay, bx = _scan_terms(s)
    final = s["state"].clone()
    if "offsets" in s:
        some, first, last = _starts(s)
        bx[0, first] += decay[0, first] * s["state"][some]
        decay[0, first] = 0
        h = _running(decay, bx)
        final[some] = h[0, last]
    else:
        bx[:, 0] += decay[:, 0] * s["state"]
        h = _running(decay, bx)
        final = h[:, -1].clone()
    y = (h * _per_channel(s["C"], s)).sum(-1) + s["D"] * u
    z = _f(s["z"]).reshape(u.shape)
    return [_like(y * z * torch.sigmoid(z), s), final]


def _plain_scan_train(s):
    u, raw, dt, decay, bx = _scan_terms(s)
    c = _per_channel(s["C"], s)
    a = decay
    if "offsets" in s:
        _, first, _ = _starts(s)
        a = decay.clone()
        a[0, first] = 0
    h = _running(a, bx)
    y = (h * c).sum(-1) + s["D"] * u
    z, dy = _f(s["z"]).reshape(u.shape), _f(s["grad"]).reshape(u.shape)
    sig = torch.sigmoid(z)
    ds = dy * z * sig
    # the reverse run: g_t = ds_t C_t + a_{t+1} g_{t+1}
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _running(after.flip(1), (ds[..., None] * c).flip(1)).flip(1)
    held = a * torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)  # a_t h_{t-1}
    gb = (g * _per_channel(s["B"], s)).sum(-1)
    ddt = u * gb + (g * held * s["A"]).sum(-1)
    ddelta = ddt * torch.sigmoid(raw)
    gr, n, d = s["case"]["groups"], s["case"]["states"], s["case"]["channels"]

    def of_group(x, like):
        return x.reshape(*x.shape[:2], gr, d // gr, n).sum(3).reshape(like.shape).to(like.dtype)

    return {"out": _like(y * z * sig, s), "u": _like(s["D"] * ds + dt * gb, s), "delta": _like(ddelta, s),
            "A": (g * held * dt[..., None]).sum((0, 1)), "B": of_group(g * (dt * u)[..., None], s["B"]),
            "C": of_group(ds[..., None] * h, s["C"]), "D": (ds * u).sum((0, 1)),
            "z": _like(dy * y * sig * (1 + z * (1 - sig)), s), "delta_bias": ddelta.sum((0, 1))}


def _plain_scan_step(s):
    slots = s["slots"].long()
    u = _f(s["u"])
    dt = _softplus(_f(s["delta"]) + s["delta_bias"])
    gr, n, d = s["case"]["groups"], s["case"]["states"], s["case"]["channels"]
    b, c = (_f(x).reshape(-1, gr, 1, n).expand(-1, -1, d // gr, -1).reshape(-1, d, n) for x in (s["B"], s["C"]))
    h = torch.exp(dt[..., None] * s["A"]) * s["state"][slots] + (dt * u)[..., None] * b
    new = s["state"].clone()
    new[slots] = h
    z = _f(s["z"])
    return [_like(((h * c).sum(-1) + s["D"] * u) * z * torch.sigmoid(z), s), new]


_PLAIN = {"conv": _plain_conv, "conv_train": _plain_conv_train, "conv_step": _plain_conv_step, "scan": _plain_scan,
          "scan_train": _plain_scan_train, "scan_step": _plain_scan_step}


# ---------------------------------------------------------------- 64 bits


def _spans(case, s):
    """(rows of one sequence as an index into [.., tokens, channels], its number) of each sequence."""
    if case["op"].endswith("step"):
        return []
    if not case["tokens"]:
        return [((slice(None),), None)]
    at = s["offsets"].tolist()
    return [((slice(at[i], at[i + 1]),), i) for i in range(case["batch"]) if at[i + 1] > at[i]]


def exact(case, seed):
    """The definition, token after token, in 64 bits; sequences of a dense call
    side by side, packed ones one after another."""
    s = _inputs(case, seed)
    steps = sum(1 for _ in _spans(case, s)) and (case["tokens"] or case["length"])
    if steps > 30000:
        return None
    s = {k: v.double() if v.is_floating_point() else v for k, v in s.items()}
    return _exact_conv(case, s) if case["op"].startswith("conv") else _exact_scan(case, s)


def _exact_conv(case, s):
    w, x, wt = case["width"], s["x"], s["weight"]
    if case["op"] == "conv_step":
        new, out = s["state"].clone(), torch.zeros_like(x)
        slots = s["slots"].long()
        held = s["state"][slots]
        p = s["bias"] + x * wt[:, w - 1]
        for k in range(w - 1):
            p = p + held[:, k] * wt[:, k]
        new[slots, :-1] = held[:, 1:]
        new[slots, -1] = x
        out = p / (1 + torch.exp(-p))
        return [out, new]
    train = case["op"] == "conv_train"
    out, final = torch.zeros_like(x), s["state"].clone()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(wt), torch.zeros_like(s["bias"])
    for at, i in _spans(case, s):
        seq = x if i is None else x[at][None]  # [sequences, tokens, channels]
        st = s["state"] if i is None else s["state"][i][None]
        n = seq.shape[1]
        padded = torch.cat([st * 0 if train else st, seq], 1)
        p = s["bias"].expand_as(seq).clone()
        for k in range(w):
            p += padded[:, k:k + n] * wt[:, k]
        sig = 1 / (1 + torch.exp(-p))
        y = p * sig
        if train:
            dp = s["grad"] if i is None else s["grad"][at][None]
            dp = dp * (sig + y * (1 - sig))
            back = torch.zeros_like(padded)
            for k in range(w):
                back[:, k:k + n] += dp * wt[:, k]
                dw[:, k] += (dp * padded[:, k:k + n]).sum((0, 1))
            db += dp.sum((0, 1))
        if i is None:
            out, final = y, padded[:, n:]
            dx = back[:, w - 1:] if train else dx
        else:
            out[at], final[i] = y[0], padded[0, n:]
            if train:
                dx[at] = back[0, w - 1:]
    return {"out": out, "x": dx, "weight": dw, "bias": db} if train else [out, final]


def _exact_scan(case, s):
    gr, n, d = case["groups"], case["states"], case["channels"]
    train, step = case["op"] == "scan_train", case["op"] == "scan_step"
    raw = s["delta"] + s["delta_bias"]
    dt = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30))))
    gate = 1 / (1 + torch.exp(-s["z"]))
    u, a_, skip = s["u"], s["A"], s["D"]

    def wide(x):  # one token's [sequences, groups * states] to [sequences, channels, states]
        return x.reshape(-1, gr, n).repeat_interleave(d // gr, 1)

    if step:
        slots = s["slots"].long()
        h = torch.exp(dt[..., None] * a_) * s["state"][slots] + (dt * u)[..., None] * wide(s["B"])
        new = s["state"].clone()
        new[slots] = h
        return [((h * wide(s["C"])).sum(-1) + skip * u) * s["z"] * gate, new]
    out, final = torch.zeros_like(u), s["state"].clone()
    grads = {k: torch.zeros_like(s[k]) for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")}
    for at, i in _spans(case, s):
        part = {k: (s[k] if i is None else s[k][at][None]) for k in ("u", "z", "B", "C")}
        q, sg = (x if i is None else x[at][None] for x in (dt, gate))
        h = s["state"] if i is None else s["state"][i][None]
        h = h * 0 if train else h
        kept, y = [], torch.zeros_like(part["u"])
        for t in range(q.shape[1]):
            if train:
                kept.append(h)
            h = torch.exp(q[:, t, :, None] * a_) * h + (q[:, t] * part["u"][:, t])[..., None] * wide(part["B"][:, t])
            y[:, t] = (h * wide(part["C"][:, t])).sum(-1) + skip * part["u"][:, t]
        last = h
        if train:
            dy = s["grad"] if i is None else s["grad"][at][None]
            ds = dy * part["z"] * sg
            sub = {k: torch.zeros_like(part["u"]) for k in ("u", "delta")}
            db, dc = torch.zeros_like(part["B"]), torch.zeros_like(part["C"])
            carry = torch.zeros_like(h)
            for t in range(q.shape[1] - 1, -1, -1):
                b, c = wide(part["B"][:, t]), wide(part["C"][:, t])
                decay = torch.exp(q[:, t, :, None] * a_)
                xt = part["u"][:, t]
                held = decay * kept[t]
                now = held + (q[:, t] * xt)[..., None] * b
                carry = carry + ds[:, t, :, None] * c
                gb = (carry * b).sum(-1)
                sub["u"][:, t] = skip * ds[:, t] + q[:, t] * gb
                sub["delta"][:, t] = xt * gb + (carry * held * a_).sum(-1)
                grads["A"] += (carry * held * q[:, t, :, None]).sum(0)
                db[:, t] = (carry * (q[:, t] * xt)[..., None]).reshape(-1, gr, d // gr, n).sum(2).flatten(1)
                dc[:, t] = (ds[:, t, :, None] * now).reshape(-1, gr, d // gr, n).sum(2).flatten(1)
                carry = carry * decay
            sub["delta"] = sub["delta"] / (1 + torch.exp(-(raw if i is None else raw[at][None])))
            sub["z"] = dy * y * sg * (1 + part["z"] * (1 - sg))
            grads["D"] += (ds * part["u"]).sum((0, 1))
            grads["delta_bias"] += sub["delta"].sum((0, 1))
            sub["B"], sub["C"] = db, dc
            for k, v in sub.items():
                if i is None:
                    grads[k] = v
                else:
                    grads[k][at] = v[0]
        y = y * part["z"] * sg
        if i is None:
            out, final = y, last
        else:
            out[at], final[i] = y[0], last[0]
    return {"out": out, **grads} if train else [out, final]


# ---------------------------------------------------------------- the work


def work(case):
    """Each input read and each output written once; the operations of the
    formulas: 2 per tap and about 8 for an activation, 7 per state and token
    (the product of the time step and A, the exponential, the input's product,
    two multiply-adds), 14 more for its gradients."""
    e, d, b = BYTES[case["dtype"]], case["channels"], case["batch"]
    op = case["op"]
    rows = b if op.endswith("step") else case["tokens"] or b * case["length"]
    if op.startswith("conv"):
        w = case["width"]
        state = 2 * b * (w - 1) * d * e
        if op == "conv_train":
            return {"bytes": 4 * e * rows * d + 8 * d * (w + 1), "flops": rows * d * (6 * w + 24)}
        return {"bytes": 2 * e * rows * d + state + 4 * d * (w + 1), "flops": rows * d * (2 * w + 8)}
    n, gr = case["states"], case["groups"]
    params = 4 * d * (n + 2)
    if op == "scan_train":
        # u, delta, z, the output's gradient; the output and three gradients
        return {"bytes": 8 * e * rows * d + 4 * e * rows * gr * n + 2 * params, "flops": rows * d * (21 * n + 60)}
    return {"bytes": 4 * e * rows * d + 2 * e * rows * gr * n + params + 8 * b * d * n,
            "flops": rows * d * (7 * n + 24)}
