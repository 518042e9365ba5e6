"""The gated linear recurrence on the GPU against the 64-bit oracle: forward,
backward and single tokens; sizes, layouts, packed sequences, options.

Tolerances.  u = 2^-24.  The kernel's a has a relative error of at most 16 u
|log a| + 2 u (exponent: the gate's argument, exponential, sum and reciprocal and the
decay's softplus; the exponential itself) and m i x one of 40 u.  A state is a sum
of such terms times products of at most L shares, the errors of which add up to 16 u |log
a| + 2 u for each of them; the sum of |log a| behind a term that still matters is
small against L, and never above the 88 that leave nothing of it.  That is (40 + 16 *
88 / 8 + 4 L) u, the eighth since a product e^-s has s e^-s < 0.4 of its error, below
(240 + 4 L) u of the sum of the terms' absolute values; gradients go by two such sums,
twice that.  Rows are then rounded by half a step of their type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import ferrum_gpu
from ferrum_gpu import ssm
from gpu_tensor import Gpu, fill, like, room, same, up, use, values
import rec_oracle as oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


@pytest.fixture(autouse=True)
def on_device(gpu_device):
    yield from use(gpu_device)


def inputs(lead, channels, dtype, seed=0, layout="plain"):
    """CPU tensors in the rows' type; "windows": columns of wider arrays."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    t = TYPES[dtype]
    if layout == "windows":
        pad = 8 if channels % 8 == 0 else 3
        wide = n(*lead, 3 * (channels + pad)).to(t)
        parts = [wide[..., k * (channels + pad):k * (channels + pad) + channels] for k in range(3)]
    else:
        parts = [n(*lead, channels).to(t) for _ in range(3)]
    x, ga, gx = parts
    return {"x": x, "gate_a": ga, "gate_x": gx, "decay": torch.linspace(-9, 1, channels) + 0.3 * n(channels),
            "bias_a": 0.5 * n(channels), "bias_x": 0.5 * n(channels)}


def spans_of(lead, offsets):
    """Rows of each sequence in [rows, channels] of all."""
    if offsets is None:
        return [range(s * lead[1], (s + 1) * lead[1]) for s in range(lead[0])]
    at = [min(max(int(v), 0), lead[0]) for v in offsets]
    return [range(at[s], at[s + 1]) for s in range(len(at) - 1)]


def d64(x, channels):
    return torch.zeros(channels, dtype=torch.float64) if x is None else x.double()


def oracle_of(v, rate, lead, offsets=None, initial=None, grad=None, grad_final=None):
    """Outputs [rows, channels] (NaN in rows of no sequence), states, gradients and their sizes, all sequences."""
    ch = v["x"].shape[-1]
    flat = {k: v[k].double().reshape(-1, ch) for k in ("x", "gate_a", "gate_x")}
    spans = spans_of(lead, offsets)
    out = torch.full_like(flat["x"], float("nan"))
    size, final = out.clone(), torch.zeros(len(spans), ch, dtype=torch.float64)
    g = {k: torch.full_like(out, float("nan")) for k in ("x", "gate_a", "gate_x")}
    by = {k: t.clone() for k, t in g.items()}
    for k in ("decay", "bias_a", "bias_x"):
        g[k], by[k] = torch.zeros(ch, dtype=torch.float64), torch.zeros(ch, dtype=torch.float64)
    g["initial"], by["initial"] = torch.zeros_like(final), torch.zeros_like(final)
    p = [d64(v[k], ch) for k in ("decay", "bias_a", "bias_x")]
    for s, rows in enumerate(spans):
        at = slice(rows.start, rows.stop)
        args = (flat["x"][at], flat["gate_a"][at], flat["gate_x"][at], *p, rate)
        h0 = d64(None if initial is None else initial[s], ch)
        out[at], _, final[s] = oracle.forward(*args, h0)
        size[at], _, _ = oracle.forward(args[0].abs(), *args[1:], h0.abs())
        if grad is not None:
            gf = d64(None if grad_final is None else grad_final[s], ch)
            gs, bs = oracle.backward(*args, h0, grad.double().reshape(-1, ch)[at], gf)
            for k in gs:
                if k == "initial":
                    g[k][s], by[k][s] = gs[k], bs[k]
                elif k in ("decay", "bias_a", "bias_x"):
                    g[k] += gs[k]
                    by[k] += bs[k]
                else:
                    g[k][at], by[k][at] = gs[k], bs[k]
    return out, size, final, g, by


def close(got, want, size, tokens, what, dtype="float32", twice=1):
    """Rows of no sequence (NaN in `want`) hold what was in them before, 7."""
    got = values(got).reshape(want.shape)
    want, size = want.numpy(), size.numpy()
    none = np.isnan(want)
    assert np.all(got[none] == 7), f"{what}: rows of no sequence were written"
    step = 0 if dtype == "float32" else torch.finfo(TYPES[dtype]).eps / 2
    least = 0 if dtype == "float32" else torch.finfo(TYPES[dtype]).tiny * torch.finfo(TYPES[dtype]).eps
    # the size's largest of a channel: errors of a state reach all tokens behind it
    top = np.max(np.where(none, 0, size), axis=0, initial=0) if size.ndim == 2 else size
    bound = np.broadcast_to(twice * (240 + 4 * tokens) * U * top, want.shape)
    bound = bound + step * (np.abs(want) + bound) + least + 1e-37
    off = np.abs(got - want)
    bad = ~none & ~(off <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} values off, worst {np.nanmax((off / bound)[~none]):.2f} times the bound"


def run(dev, lead, channels, dtype, rate=8.0, layout="plain", offsets=None, bias=True, state=True, tokens=None,
        backward=True, length=None, seed=0):
    v = inputs(lead, channels, dtype, seed, layout)
    if not bias:
        v["bias_a"] = v["bias_x"] = None
    batch = lead[0] if offsets is None else len(offsets) - 1
    g = torch.Generator().manual_seed(seed + 1)
    initial = torch.randn(batch, channels, generator=g) if state else None
    grad = torch.randn(*lead, channels, generator=g).to(TYPES[dtype])
    grad_final = torch.randn(batch, channels, generator=g) if state else None
    plan = ssm.RecurrencePlan(batch, lead[1] if offsets is None else (length or lead[0]), channels, dev, dtype=dtype,
                              rate=rate, tokens=lead[0] if offsets is not None else None)
    at = None if offsets is None else up(torch.tensor(offsets, dtype=torch.int32))
    d = {k: up(t) for k, t in v.items()}
    out, final = fill((*lead, channels), dtype), fill((batch, channels))
    check = room(plan.checkpoint_bytes)
    kw = {"bias_a": d["bias_a"], "bias_x": d["bias_x"], "offsets": at}
    plan.forward(d["x"], d["gate_a"], d["gate_x"], d["decay"], out, initial=up(initial), final=final,
                 checkpoints=check, **kw)
    longest = max((len(s) for s in spans_of(lead, offsets)), default=0)
    want, size, last, g64, by = oracle_of(v, rate, lead, offsets, initial, grad, grad_final)
    close(out, want, size, longest, "out", dtype)
    close(final, last, size.nan_to_num(0).max(0).values.expand_as(last) + (0 if initial is None else initial.abs()),
          longest, "final")
    if backward:
        names = {k: fill((*lead, channels), dtype) for k in ("x", "gate_a", "gate_x")}
        names |= {k: fill((channels,)) for k in ("decay", "bias_a", "bias_x")}
        names["initial"] = fill((batch, channels))
        plan.backward(d["x"], d["gate_a"], d["gate_x"], d["decay"], up(grad), check, grad_final=up(grad_final), **kw,
                      **{"grad_" + k: t for k, t in names.items()})
        for k, t in names.items():
            close(t, g64[k], by[k], longest, "gradient of " + k,
                  dtype if k in ("x", "gate_a", "gate_x") else "float32", twice=2)
    plan.destroy()


@pytest.mark.parametrize("batch,length,channels,dtype", [
    (1, 1, 1, "float32"), (2, 3, 5, "bfloat16"), (1, 7, 64, "float16"), (3, 8, 68, "bfloat16"),
    (1, 31, 130, "float32"), (2, 33, 64, "bfloat16"), (1, 127, 66, "float16"), (1, 128, 64, "float32"),
    (1, 129, 192, "bfloat16"), (2, 255, 100, "float16"), (1, 256, 64, "bfloat16"), (1, 257, 61, "bfloat16"),
    (5, 513, 64, "bfloat16"), (1, 1025, 70, "float16"), (2, 1000, 128, "float32"), (1, 2049, 260, "bfloat16"),
    (1, 5003, 64, "bfloat16"), (3, 2600, 130, "float32")])
def test_sizes(gpu_device, batch, length, channels, dtype):
    run(gpu_device, (batch, length), channels, dtype)


@pytest.mark.parametrize("layout,channels", [("windows", 64), ("windows", 37), ("plain", 64)])
@pytest.mark.parametrize("bias,state", [(True, False), (False, True), (False, False)])
def test_layouts_and_options(gpu_device, layout, channels, bias, state):
    run(gpu_device, (2, 300), channels, "bfloat16", layout=layout, bias=bias, state=state)


@pytest.mark.parametrize("rate", [0.0, 0.5, 64.0])
def test_rates(gpu_device, rate):
    """0: nothing decays and nothing enters."""
    run(gpu_device, (1, 200), 64, "float32", rate=rate, backward=rate > 0)


@pytest.mark.parametrize("dtype,channels", [("float32", 64), ("bfloat16", 96), ("float16", 61)])
@pytest.mark.parametrize("offsets", [
    [0, 1, 2, 3, 4, 5, 6, 7, 8, 9], [0, 300, 300, 310, 700], [0, 0, 0, 5, 5, 133, 133], [3, 10, 10, 140, 500],
    [0, 8, 16, 24, 32, 64, 128, 256, 512], [0, 256, 512, 768], [5, 5, 5], [0, 33, 990, 990]])
def test_packed(gpu_device, dtype, channels, offsets):
    """Short and long sequences, empty ones at both ends, rows before and behind all of them."""
    run(gpu_device, (offsets[-1] + 9,), channels, dtype, offsets=offsets)


def test_packed_many(gpu_device):
    g = np.random.default_rng(0)
    lengths = g.choice([0, 1, 2, 3, 7, 40, 150], 200)
    run(gpu_device, (int(lengths.sum()),), 64, "bfloat16", offsets=[0, *np.cumsum(lengths).tolist()])


def test_offsets_beyond_the_rows_are_taken_as_the_nearest(gpu_device):
    run(gpu_device, (200,), 64, "float32", offsets=[-5, 40, 250, 300])


@pytest.mark.parametrize("packed", [False, True])
def test_no_tokens(gpu_device, packed):
    """The last state is the first one, the first one's gradient the last one's; the parameters' are 0."""
    batch, ch = 3, 70
    plan = ssm.RecurrencePlan(batch, 0, ch, gpu_device, dtype="float32", tokens=0 if packed else None)
    lead = (0,) if packed else (batch, 0)
    x = fill((*lead, ch))
    p, initial, final, back = fill((ch,), value=0.5), Gpu(torch.randn(batch, ch)), fill((batch, ch)), fill((batch, ch))
    at = Gpu(torch.zeros(batch + 1, dtype=torch.int32)) if packed else None
    check = room(plan.checkpoint_bytes)
    plan.forward(x, x, x, p, x, initial=initial, final=final, offsets=at, checkpoints=check)
    assert same(initial, final)
    sums = [fill((ch,)) for _ in range(3)]
    plan.backward(x, x, x, p, x, check, grad_final=initial, grad_initial=back, offsets=at, grad_decay=sums[0],
                  grad_bias_a=sums[1], grad_bias_x=sums[2])
    assert same(back, initial) and all((s == 0).all() for s in sums)


@pytest.mark.parametrize("batch,channels,dtype", [(1, 64, "float32"), (3, 2048, "bfloat16"), (70, 61, "float16"),
                                                  (256, 132, "bfloat16"), (5, 1, "float32")])
def test_step(gpu_device, batch, channels, dtype):
    """One token of each row, states in slots; rows without one get zeros and leave the states."""
    v = inputs((batch,), channels, dtype, layout="windows")
    rows = batch + 3
    state = torch.randn(rows, channels)
    slots = torch.randperm(rows)[:batch].to(torch.int32)
    if batch > 2:
        slots[1], slots[2] = -1, rows
    out, new = fill((batch, channels), dtype), fill((rows, channels))
    d = {k: up(t) for k, t in v.items()}
    ssm.recurrence_step(gpu_device, **d, state=up(state), out=out, slots=up(slots), state_out=new)
    inplace = up(state)
    again = fill((batch, channels), dtype)
    ssm.recurrence_step(gpu_device, **d, state=inplace, out=again, slots=up(slots))
    want, left = torch.zeros(batch, channels, dtype=torch.float64), torch.full((rows, channels), 7.0).double()
    size = want.clone()
    kept = state.double()
    for b in range(batch):
        s = int(slots[b])
        if not 0 <= s < rows:
            continue
        args = [v[k][b:b + 1].double() for k in ("x", "gate_a", "gate_x")] + \
               [v[k].double() for k in ("decay", "bias_a", "bias_x")]
        want[b], _, _ = (t[0] for t in oracle.forward(*args, 8.0, state[s].double()))
        size[b] = oracle.forward(args[0].abs(), *args[1:], 8.0, state[s].abs().double())[0][0]
        left[s] = kept[s] = want[b]
    close(out, want, size, 1, "out", dtype)
    assert same(out, again)
    got = values(new)
    moved = (left != 7).numpy()
    assert (got[~moved] == 7).all()
    assert np.abs(got - left.numpy())[moved].max() <= 250 * U * max(1, float(size.max()))
    assert np.array_equal(values(inplace)[~moved], state.double().numpy()[~moved])
    assert np.abs(values(inplace) - kept.numpy()).max() <= 250 * U * max(1, float(size.max()))


def test_step_without_slots(gpu_device):
    v = inputs((4,), 64, "float32")
    state, out = torch.randn(4, 64), fill((4, 64))
    d = {k: up(t) for k, t in v.items()}
    s = up(state)
    ssm.recurrence_step(gpu_device, d["x"], d["gate_a"], d["gate_x"], d["decay"], s, out)
    assert same(s, out)


@pytest.mark.parametrize("dtype,channels", [("float32", 64), ("bfloat16", 30)])
def test_prompt_then_tokens(gpu_device, dtype, channels):
    """A prompt's last state and single tokens behind it give what the whole sequence gives."""
    n, more = 70, 5
    v = inputs((2, n + more), channels, dtype)
    d = {k: up(t) for k, t in v.items()}
    whole, state = fill((2, n + more, channels), dtype), fill((2, channels))
    p = lambda k: {"bias_a": d["bias_a"], "bias_x": d["bias_x"], **k}  # noqa: E731
    ssm.RecurrencePlan(2, n + more, channels, gpu_device, dtype=dtype).forward(
        d["x"], d["gate_a"], d["gate_x"], d["decay"], whole, **p({}))
    cut = [d[k][:, :n] for k in ("x", "gate_a", "gate_x")]
    ssm.RecurrencePlan(2, n, channels, gpu_device, dtype=dtype).forward(*cut, d["decay"], fill((2, n, channels), dtype),
                                                                       final=state, **p({}))
    step = 8 * (torch.finfo(TYPES[dtype]).eps / 2 if dtype != "float32" else (240 + 4 * (n + more)) * U)
    for t in range(n, n + more):
        out = fill((2, channels), dtype)
        ssm.recurrence_step(gpu_device, *[d[k][:, t] for k in ("x", "gate_a", "gate_x")], d["decay"], state, out, **p({}))
        a, b = values(out), values(whole)[:, t]
        assert np.abs(a - b).max() <= step * max(1, np.abs(values(whole)).max())


@pytest.mark.parametrize("packed,length", [(False, 40), (False, 1500), (True, 700)])
def test_final_may_be_initial(gpu_device, packed, length):
    batch, ch = 3, 64
    offsets = [0, 1, 1, length] if packed else None
    lead = (length,) if packed else (batch, length)
    v = inputs(lead, ch, "float32")
    d = {k: up(t) for k, t in v.items()}
    at = up(torch.tensor(offsets, dtype=torch.int32)) if packed else None
    plan = ssm.RecurrencePlan(batch, length, ch, gpu_device, dtype="float32", tokens=length if packed else None)
    initial = torch.randn(batch, ch)
    apart, one = fill((batch, ch)), up(initial)
    outs = [fill((*lead, ch)) for _ in range(2)]
    args = (d["x"], d["gate_a"], d["gate_x"], d["decay"])
    plan.forward(*args, outs[0], initial=up(initial), final=apart, offsets=at)
    plan.forward(*args, outs[1], initial=one, final=one, offsets=at)
    assert same(apart, one) and same(*outs)


@pytest.mark.parametrize("packed", [False, True])
def test_same_bits_again(gpu_device, packed):
    lead, ch = ((2300,), 100) if packed else ((2, 1100), 100)
    offsets = [0, 700, 2300] if packed else None
    v = inputs(lead, ch, "bfloat16")
    d = {k: up(t) for k, t in v.items()}
    at = up(torch.tensor(offsets, dtype=torch.int32)) if packed else None
    plan = ssm.RecurrencePlan(2, 1600, ch, gpu_device, tokens=2300 if packed else None) if packed else \
        ssm.RecurrencePlan(2, 1100, ch, gpu_device)
    args, grad = (d["x"], d["gate_a"], d["gate_x"], d["decay"]), like(v["x"]).normal_()
    seen = None
    for _ in range(4):
        out, check = like(v["x"]), room(plan.checkpoint_bytes)
        g = {k: like(t) for k, t in v.items()}
        plan.forward(*args, out, checkpoints=check, offsets=at)
        plan.backward(*args, grad, check, offsets=at, **{"grad_" + k: t for k, t in g.items()})
        now = [t.get() for t in (out, *g.values())]
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, now))
        seen = now


def test_gradient_is_the_difference(gpu_device):
    """Differences of the loss in 64 bits of outputs in 32: (f(x + e d) - f(x - e d)) / 2e along random directions d.
    The loss is linear in outputs that are off by 500 u of their sizes, and the difference's own error is e^2 / 6 of a third
    derivative: with e = 2^-7, 1e-2 of the gradient's length covers both."""
    lead, ch, e = (2, 50), 64, 2.0 ** -7
    v = inputs(lead, ch, "float32")
    v["decay"] = torch.linspace(-5, 0, ch)
    grad = torch.randn(*lead, ch)
    plan = ssm.RecurrencePlan(*lead, ch, gpu_device, dtype="float32")
    check, out = room(plan.checkpoint_bytes), fill((*lead, ch))

    def call(w):
        d = {k: up(t) for k, t in w.items()}
        plan.forward(d["x"], d["gate_a"], d["gate_x"], d["decay"], out, bias_a=d["bias_a"], bias_x=d["bias_x"],
                     checkpoints=check)
        return (out.get().double() * grad.double()).sum().item(), d

    _, d = call(v)
    g = {k: like(t) for k, t in v.items()}
    plan.backward(d["x"], d["gate_a"], d["gate_x"], d["decay"], up(grad), check, bias_a=d["bias_a"],
                  bias_x=d["bias_x"], **{"grad_" + k: t for k, t in g.items()})
    for k in v:
        along = g[k].get()
        along = along / along.norm()
        there = [call({**v, k: v[k] + s * e * along})[0] for s in (1, -1)]
        slope = (there[0] - there[1]) / (2 * e)
        assert abs(slope / g[k].get().double().norm().item() - 1) < 1e-2, k


def test_gradients_asked_for_one_by_one(gpu_device):
    lead, ch = (2, 130), 64
    v = inputs(lead, ch, "bfloat16")
    d = {k: up(t) for k, t in v.items()}
    plan = ssm.RecurrencePlan(*lead, ch, gpu_device)
    args, check, grad = (d["x"], d["gate_a"], d["gate_x"], d["decay"]), room(plan.checkpoint_bytes), like(v["x"]).normal_()
    plan.forward(*args, like(v["x"]), checkpoints=check)
    every = {k: like(t) for k, t in v.items()}
    plan.backward(*args, grad, check, **{"grad_" + k: t for k, t in every.items()})
    for k in v:
        one = like(v[k])
        plan.backward(*args, grad, check, **{"grad_" + k: one})
        assert same(one, every[k]), k


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_nothing_leaks(gpu_device, dtype):
    """NaN and infinities of one sequence stay in it, of one channel in that; of rows outside in those."""
    offsets, n, ch = [2, 200, 200, 201, 560], 570, 64
    v = inputs((n,), ch, dtype)
    clean = {k: t.clone() for k, t in v.items()}
    initial = torch.randn(4, ch)
    bad_initial = initial.clone()
    bad_initial[1] = float("nan")   # an empty sequence's
    bad_initial[2, 5] = float("inf")
    for k in ("x", "gate_a", "gate_x"):
        v[k][:2] = float("nan")
        v[k][560:] = float("inf")
    v["x"][100, 3] = float("nan")
    v["gate_a"][150, 7] = float("nan")
    grad = torch.randn(n, ch).to(TYPES[dtype])
    bad_grad = grad.clone()
    bad_grad[:2], bad_grad[560:], bad_grad[300, 11] = float("nan"), float("nan"), float("nan")
    plan = ssm.RecurrencePlan(4, n, ch, gpu_device, dtype=dtype, tokens=n)
    at = up(torch.tensor(offsets, dtype=torch.int32))

    def call(w, h0, g):
        d = {k: up(t) for k, t in w.items()}
        out, final, check, back = fill((n, ch), dtype), fill((4, ch)), room(plan.checkpoint_bytes), fill((4, ch))
        gs = {k: fill((n, ch), dtype) for k in ("x", "gate_a", "gate_x")}
        plan.forward(d["x"], d["gate_a"], d["gate_x"], d["decay"], out, initial=up(h0), final=final, offsets=at,
                     checkpoints=check)
        plan.backward(d["x"], d["gate_a"], d["gate_x"], d["decay"], up(g), check, offsets=at, grad_initial=back,
                      **{"grad_" + k: t for k, t in gs.items()})
        return [values(t) for t in (out, final, back, *gs.values())]

    good, bad = call(clean, initial, grad), call(v, bad_initial, bad_grad)
    touched = np.zeros((n, ch), bool)   # sequence and channel of what is bad
    touched[2:200, [3, 7]] = True
    touched[200:201, 5] = True
    touched[201:560, 11] = True
    for a, b in zip((good[0], *good[3:]), (bad[0], *bad[3:])):
        assert np.array_equal(a[~touched], b[~touched])
    assert np.isnan(bad[0][100:200, 3]).all() and np.isnan(bad[0][150:200, 7]).all()
    assert np.isinf(bad[0][200, 5]) and np.isfinite(bad[0][:100, 3].sum())
    assert np.isnan(bad[3][201:301, 11]).all()
    seq = np.ones((4, ch), bool)
    seq[0, [3, 7]] = seq[2, 5] = seq[3, 11] = False
    seq[1] = False
    for a, b in zip(good[1:3], bad[1:3]):
        assert np.array_equal(a[seq], b[seq])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_extreme_gates(gpu_device, dtype):
    """Gates far open and far closed, infinite ones, decays that leave all or nothing: as the oracle, no NaN."""
    lead, ch = (1, 300), 64
    v = inputs(lead, ch, dtype)
    far = torch.tensor([-1e4, -200.0, -100.0, -80.0, 80.0, 100.0, 1e4, float("inf"), -float("inf")]).to(TYPES[dtype])
    pick = torch.randint(0, 2 * len(far), (*lead, ch))
    v["gate_a"] = torch.where(pick < len(far), far[pick % len(far)], v["gate_a"])
    pick = torch.randint(0, 2 * len(far), (*lead, ch))
    v["gate_x"] = torch.where(pick < len(far), far[pick % len(far)], v["gate_x"])
    v["decay"] = torch.linspace(-80, 12, ch)
    v["bias_a"] = v["bias_x"] = None
    initial, grad = torch.randn(1, ch), torch.randn(*lead, ch).to(TYPES[dtype])
    plan = ssm.RecurrencePlan(*lead, ch, gpu_device, dtype=dtype)
    d = {k: up(t) for k, t in v.items()}
    out, check = fill((*lead, ch), dtype), room(plan.checkpoint_bytes)
    plan.forward(d["x"], d["gate_a"], d["gate_x"], d["decay"], out, initial=up(initial), checkpoints=check)
    want, size, _, g64, by = oracle_of(v, 8.0, lead, None, initial, grad)
    close(out, want, size, 300, "out", dtype)
    g = {k: fill((*lead, ch), dtype) for k in ("x", "gate_a", "gate_x")}
    plan.backward(d["x"], d["gate_a"], d["gate_x"], d["decay"], up(grad), check,
                  **{"grad_" + k: t for k, t in g.items()})
    for k, t in g.items():
        close(t, g64[k], by[k], 300, "gradient of " + k, dtype, twice=2)


@pytest.mark.parametrize("length", [40, 2500])
def test_infinite_states_stay(gpu_device, length):
    """An infinite state stays one, however small the product of what is kept of it."""
    ch = 64
    v = inputs((1, length), ch, "float32")
    v["decay"][:] = 0.0
    d = {k: up(t) for k, t in v.items()}
    initial, out = torch.zeros(1, ch), fill((1, length, ch))
    initial[0, 1], initial[0, 2] = float("inf"), -float("inf")
    ssm.RecurrencePlan(1, length, ch, gpu_device, dtype="float32").forward(
        d["x"], d["gate_a"], d["gate_x"], d["decay"], out, initial=up(initial))
    got = values(out)
    assert (got[0, :, 1] == np.inf).all() and (got[0, :, 2] == -np.inf).all() and np.isfinite(got[0, :, 3:]).all()


def test_broadcast_inputs(gpu_device):
    """Strides of 0 for sequences and rows of inputs."""
    ch = 64
    v = inputs((1, 200), ch, "float32")
    row = torch.randn(1, 1, ch)
    plan = ssm.RecurrencePlan(3, 200, ch, gpu_device, dtype="float32")
    outs = [fill((3, 200, ch)) for _ in range(2)]
    x, gx = up(v["x"]), up(row)
    plan.forward(x.expand(3, 200, ch), x.expand(3, 200, ch), gx.expand(3, 200, ch), up(v["decay"]), outs[0])
    full = [up(t.expand(3, 200, ch).contiguous()) for t in (v["x"], v["x"], row.expand(1, 200, ch))]
    plan.forward(*full, up(v["decay"]), outs[1])
    assert same(*outs)


def test_device_buffers_and_addresses(gpu_device):
    lead, ch = (2, 70), 64
    v = inputs(lead, ch, "float32")
    d = {k: up(t) for k, t in v.items()}
    plan = ssm.RecurrencePlan(*lead, ch, gpu_device, dtype="float32")
    outs = [fill((*lead, ch)) for _ in range(2)]
    plan.forward(d["x"], d["gate_a"], d["gate_x"], d["decay"], outs[0])
    plan.forward(d["x"].buf, d["gate_a"].data_ptr(), d["gate_x"].buf, d["decay"].buf, outs[1].data_ptr())
    assert same(*outs)
    small = ferrum_gpu.hip.DeviceBuffer(gpu_device, 64)
    with pytest.raises(ValueError, match="buffer of 64 bytes"):
        plan.forward(small, d["gate_a"], d["gate_x"], d["decay"], outs[1])


@pytest.mark.parametrize("packed", [False, True])
def test_captured_calls_replay(gpu_device, packed):
    """Forward, backward and a step in a graph, replayed on changing inputs with eager work between."""
    n, ch = 900, 64
    lead = (n,) if packed else (2, n)
    offsets = [0, 333, n] if packed else None
    v = inputs(lead, ch, "bfloat16")
    d = {k: up(t) for k, t in v.items()}
    at = up(torch.tensor(offsets, dtype=torch.int32)) if packed else None
    plan = ssm.RecurrencePlan(2, n, ch, gpu_device, tokens=n if packed else None)
    out, check, grad = like(v["x"]), room(plan.checkpoint_bytes), like(v["x"]).normal_()
    g = {k: like(t) for k, t in v.items()}
    token, state, stepped = Gpu(torch.randn(2, ch).bfloat16()), Gpu(torch.zeros(2, ch)), Gpu(torch.zeros(2, ch).bfloat16())
    args = (d["x"], d["gate_a"], d["gate_x"], d["decay"])

    def calls(stream=0):
        plan.forward(*args, out, offsets=at, checkpoints=check, stream=stream)
        plan.backward(*args, grad, check, offsets=at, stream=stream, **{"grad_" + k: t for k, t in g.items()})
        ssm.recurrence_step(gpu_device, token, token, token, d["decay"], state, stepped, stream=stream)

    with pytest.raises(ferrum_gpu._native.FerrumGpuError, match="first backward call"):
        with ferrum_gpu.hip.Capture(gpu_device) as cap:
            plan.backward(*args, grad, check, offsets=at, stream=cap.stream)
    calls()
    gpu_device.sync()
    with ferrum_gpu.hip.Capture(gpu_device, keep=[plan, args, out, check, grad, g, token, state, stepped]) as cap:
        calls(cap.stream)
    for k in range(4):
        for t in (d["x"], grad, token):
            t.normal_()
        before = state.clone()
        cap.graph.launch()
        gpu_device.sync()
        replayed = [t.get() for t in (out, *g.values(), state, stepped)]
        state.copy_(before)
        calls()
        assert all(torch.equal(a, b) for a, b in zip(replayed, [t.get() for t in (out, *g.values(), state, stepped)])), k


def test_refusals(gpu_device):
    lead, ch = (2, 16), 64
    plan = ssm.RecurrencePlan(*lead, ch, gpu_device, dtype="float32")
    x, p, out = fill((*lead, ch)), fill((ch,)), fill((*lead, ch))
    error = ferrum_gpu._native.FerrumGpuError
    for bad, why in ((dict(x=fill((2, 15, ch))), "shape"), (dict(gate_a=fill((*lead, ch), "bfloat16")), "bfloat16"),
                     (dict(decay=fill((ch + 1,))), "shape"), (dict(offsets=fill((3,), "int32", 0)), "offsets"),
                     (dict(initial=fill((2, ch + 1))), "shape"), (dict(checkpoints=room(8)), "contiguous bytes")):
        with pytest.raises(ValueError, match=why):
            plan.forward(**{**dict(x=x, gate_a=x, gate_x=x, decay=p, out=out), **bad})
    for bad, why in ((dict(out=x), "overlap"), (dict(out=0), "null buffer"), (dict(decay=0), "null buffer"),
                     (dict(final=x.data_ptr()), "overlap"), (dict(x=x.data_ptr() + 2), "not aligned")):
        with pytest.raises(error, match=why):
            plan.forward(**{**dict(x=x, gate_a=x, gate_x=x, decay=p, out=out), **bad})
    check = room(plan.checkpoint_bytes)
    with pytest.raises(error, match="overlap"):
        plan.backward(x, x, x, p, x, check, grad_x=out, grad_gate_a=out)
    with pytest.raises(error, match="null buffer"):
        plan.backward(x, x, x, p, x, 0, grad_x=out)
    for bad in (dict(rate=-1.0), dict(rate=float("nan")), dict(rate=float("inf")), dict(rate=1e39),
                dict(channels=0), dict(batch=-1), dict(length=2 ** 31), dict(tokens=-1)):
        with pytest.raises(error):
            ssm.RecurrencePlan(**{**dict(batch=2, length=16, channels=ch, device=gpu_device), **bad})
    with pytest.raises(error, match="state_rows"):
        ssm.recurrence_step(gpu_device, x[:, 0], x[:, 0], x[:, 0], p, fill((1, ch)), out[:, 0])
    with pytest.raises(error, match="rate"):
        ssm.recurrence_step(gpu_device, x[:, 0], x[:, 0], x[:, 0], p, fill((2, ch)), out[:, 0], rate=-2)
    plan.destroy()
    with pytest.raises(ValueError, match="destroyed"):
        plan.forward(x, x, x, p, out)


def test_plans_say_how_they_run(gpu_device):
    plan = ssm.RecurrencePlan(2, 40, 64, gpu_device)
    got = plan.describe()
    assert got["forward_tokens"] >= 32 and got["backward_tokens"] >= 32


@pytest.mark.parametrize("dtype,channels", [("bfloat16", 64), ("float32", 130), ("float16", 66)])
def test_rows_at_odd_places(gpu_device, dtype, channels):
    """Rows that begin at any element give what aligned ones give, forward and backward."""
    lead = (2, 300)
    v = inputs(lead, channels, dtype)
    plan = ssm.RecurrencePlan(*lead, channels, gpu_device, dtype=dtype)
    grad, decay = torch.randn(*lead, channels).to(TYPES[dtype]), up(v["decay"])
    seen = []
    for odd in (0, 1):
        wide = lambda x: torch.nn.functional.pad(x, (odd, odd))  # noqa: E731
        cut = lambda x: x[..., odd:odd + channels]  # noqa: E731
        x, ga, gx, dy = (cut(up(wide(t))) for t in (v["x"], v["gate_a"], v["gate_x"], grad))
        outs = [fill((*lead, channels + 2 * odd), dtype) for _ in range(4)]
        check, sums = room(plan.checkpoint_bytes), fill((channels,))
        plan.forward(x, ga, gx, decay, cut(outs[0]), checkpoints=check)
        plan.backward(x, ga, gx, decay, dy, check, grad_x=cut(outs[1]), grad_gate_a=cut(outs[2]),
                      grad_gate_x=cut(outs[3]), grad_decay=sums)
        seen.append([*(cut(o).get() for o in outs), sums.get()])
        if odd:
            assert all((o.get()[..., [0, -1]] == 7).all() for o in outs)
    assert all(torch.equal(a, b) for a, b in zip(*seen))


def test_packed_sequences_of_one_token(gpu_device):
    """As many as three looks of 64 lanes find, against the single token's call; some without any."""
    n, ch = 9000, 66
    lengths = torch.ones(n, dtype=torch.int64)
    lengths[::7] = 0
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).to(torch.int32)
    rows = int(offsets[-1])
    v = inputs((rows,), ch, "float32")
    d = {k: up(t) for k, t in v.items()}
    initial = torch.randn(n, ch)
    out, final = fill((rows, ch)), fill((n, ch))
    ssm.RecurrencePlan(n, 1, ch, gpu_device, dtype="float32", tokens=rows).forward(
        d["x"], d["gate_a"], d["gate_x"], d["decay"], out, bias_a=d["bias_a"], bias_x=d["bias_x"], initial=up(initial),
        final=final, offsets=up(offsets))
    some = torch.nonzero(lengths)[:, 0]
    state, want = up(initial), fill((rows, ch))
    ssm.recurrence_step(gpu_device, **d, state=state, out=want, slots=up(some.to(torch.int32)))
    assert np.abs(values(out) - values(want)).max() <= 500 * U * 5
    assert np.abs(values(final) - values(state)).max() <= 500 * U * 5
    none = torch.nonzero(lengths == 0)[:, 0]
    assert torch.equal(final.get()[none], initial[none])


def test_rows_far_apart(gpu_device):
    """Rows whose offsets pass 32 bits: 2^25 elements between rows, 96 of them in one buffer of 6.4 GB."""
    from gpu_tensor import Far
    from ferrum_gpu.hip import DeviceBuffer
    n, ch, row = 96, 64, 1 << 25
    v = inputs((1, n), ch, "bfloat16")
    buf = DeviceBuffer(gpu_device, 2 * ((n - 1) * row + 4 * ch))
    far = [Far(buf, t, row, k * ch) for k, t in enumerate((v["x"], v["gate_a"], v["gate_x"], torch.zeros_like(v["x"])))]
    plan, decay = ssm.RecurrencePlan(1, n, ch, gpu_device), up(v["decay"])
    check, grad = room(plan.checkpoint_bytes), like(v["x"]).normal_()
    out, dx, da = like(v["x"]), like(v["x"]), like(v["x"])
    plan.forward(up(v["x"]), up(v["gate_a"]), up(v["gate_x"]), decay, out, checkpoints=check)
    plan.backward(up(v["x"]), up(v["gate_a"]), up(v["gate_x"]), decay, grad, check, grad_x=dx, grad_gate_a=da)
    plan.forward(*far[:3], decay, far[3], checkpoints=check)
    gpu_device.sync()
    assert same(out, far[3])
    ga = like(v["x"])
    plan.backward(*far[:3], decay, grad, check, grad_x=far[3], grad_gate_a=ga)
    gpu_device.sync()
    assert same(dx, far[3]) and same(da, ga)
    buf.free()
