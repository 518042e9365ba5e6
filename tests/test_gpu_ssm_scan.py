"""The selective scan on the GPU against its 64-bit oracle: whole sequences,
gradients, single tokens; layouts, packed sequences, states, refusals."""

from __future__ import annotations

import numpy as np
import pytest

import ssm_oracle as o

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import gpu_tensor  # noqa: E402
from gpu_tensor import Far, fill, like, room, same, up, values  # noqa: E402


@pytest.fixture(autouse=True)
def _on_gpu(gpu_device):
    yield from gpu_tensor.use(gpu_device)

GRADS = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")


def _type(dtype):
    return getattr(torch, dtype)


def _inputs(rng, lead, channels, states, groups, dtype, batch):
    """Inputs as a model has them; the time steps around 0.1 to 2."""
    t = lambda *s, k=1.0: (torch.from_numpy(rng.standard_normal(s)) * k).to(_type(dtype))  # noqa: E731
    f = lambda v: torch.from_numpy(v).float()  # noqa: E731
    return dict(u=t(*lead, channels), delta=t(*lead, channels, k=0.5), z=t(*lead, channels),
                B=t(*lead, groups, states), C=t(*lead, groups, states), gy=t(*lead, channels),
                A=f(-rng.uniform(0.2, 1.5, (channels, states))), D=f(rng.standard_normal(channels)),
                delta_bias=f(rng.uniform(-2.5, -0.5, channels)), initial=f(rng.standard_normal((batch, channels, states))),
                gfinal=f(rng.standard_normal((batch, channels, states))))


def _oracle_args(i, at, s, use_softplus, without):
    a = {k: values(i[k][at]) for k in ("u", "delta", "B", "C")}
    a.update(A=values(i["A"]), use_softplus=use_softplus, grad=values(i["gy"][at]))
    for name, key in (("D", "D"), ("delta_bias", "bias")):
        a[key] = None if name in without else values(i[name])
    a["z"] = None if "z" in without else values(i["z"][at])
    for name, key in (("initial", "initial"), ("gfinal", "grad_final")):
        a[key] = None if name in without else values(i[name][s])
    return a


def _compare(got, i, spans, channels, groups, states, dtype, use_softplus=True, without=()):
    """Results against the oracle's, sequence by sequence; parameters' gradients summed over them."""
    tokens = sum(len(range(*at[-1].indices(10 ** 9))) if isinstance(at, tuple) else 0 for at, _ in spans)
    total = {}
    rounds_of = {}
    for at, s in spans:
        a = _oracle_args(i, at, s, use_softplus, without)
        raw = a["delta"] + (0 if a["bias"] is None else a["bias"])
        most = float(np.abs(o.softplus(raw) if use_softplus else raw).max()) if raw.size else 0.0
        r, m = o.scan(**a), o.scan(**a, magnitude=True)
        per_token = channels // groups
        rounds = o.scan_rounds(raw.shape[0], a["A"], most, states)
        summed = o.scan_rounds(raw.shape[0], a["A"], most, states, per_token)
        o.within(values(got["out"][at]), r["out"], m["out"], rounds, dtype, "out")
        if "final" in got:
            o.within(values(got["final"][s]), r["final"], m["final"], rounds, "float32", "final")
        if "u" not in got:
            continue
        for k in ("u", "delta", "z"):
            if k in got:
                o.within(values(got[k][at]), r[k], m[k], 2 * rounds, dtype, "grad_" + k)
        for k in ("B", "C"):
            o.within(values(got[k][at]).reshape(r[k].shape), r[k], m[k], 2 * summed, dtype, "grad_" + k)
        if "initial" in got:
            o.within(values(got["initial"][s]), r["initial"], m["initial"], rounds, "float32", "grad_initial")
        for k, name in (("A", "A"), ("D", "D"), ("bias", "delta_bias")):
            x, y = total.get(name, (0, 0))
            total[name] = x + r[k], y + m[k]
            rounds_of[name] = max(rounds_of.get(name, 0), 2 * rounds)
    for name, (x, y) in total.items():
        o.within(values(got[name]), x, y, rounds_of[name] + tokens + sum(i["u"].shape[:-1]), "float32", "grad_" + name)


def _check(dev, rng, batch, length, channels, states, groups, dtype, use_softplus=True, without=(), layout="plain"):
    import ferrum_gpu
    i = _inputs(rng, (batch, length), channels, states, groups, dtype, batch)
    if not use_softplus:
        i["delta"] = i["delta"].abs() * 0.3
        i["delta_bias"] = i["delta_bias"].abs() * 0.1

    def laid(v, room=False):
        v = torch.full_like(v, 7) if room else v
        if v.dim() == 4 and layout != "plain":
            v = v.flatten(2)
        if layout == "window":
            n = v.shape[-1]
            big = torch.full(v.shape[:2] + (2 * n + 5,), 7.0, dtype=v.dtype)
            big[..., n + 3:2 * n + 3] = v
            return up(big[..., n + 3:2 * n + 3])
        if layout == "tokens":
            return up(v.transpose(0, 1).contiguous().transpose(0, 1))
        return up(v)

    d = {k: laid(v) if k in ("u", "delta", "z", "B", "C", "gy") else up(v) for k, v in i.items()}
    got = {"out": laid(i["u"], True), "final": fill(i["initial"].shape), "initial": fill(i["initial"].shape)}
    got.update({k: laid(i[k], True) if k in ("u", "delta", "z", "B", "C") else fill(i[k].shape) for k in GRADS})
    opt = {k: d[k] for k in ("D", "z", "delta_bias") if k not in without}
    if "z" in without:
        del got["z"]
    plan = ferrum_gpu.ssm.ScanPlan(batch, length, channels, states, dev, groups=groups, dtype=dtype,
                                   softplus=use_softplus)
    check = room(plan.checkpoint_bytes)
    main = [d[k] for k in ("u", "delta", "A", "B", "C")]
    plan.forward(*main, got["out"], **opt, initial=None if "initial" in without else d["initial"],
                 final=got["final"], checkpoints=check)
    plan.backward(*main, d["gy"], check, **opt, **{"grad_" + k: got[k] for k in GRADS if k in got},
                  grad_initial=got["initial"], grad_final=None if "gfinal" in without else d["gfinal"])
    dev.sync()
    at = [((s, slice(0, length)), s) for s in range(batch)]
    _compare(got, i, at, channels, groups, states, dtype, use_softplus, without)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("batch,length,channels,states,groups", [
    (1, 1, 16, 16, 1), (2, 2, 64, 16, 1), (1, 3, 1, 1, 1), (3, 15, 15, 3, 1), (2, 16, 17, 4, 1), (1, 17, 70, 5, 1),
    (2, 33, 130, 8, 2), (1, 64, 48, 13, 3), (2, 65, 64, 16, 2), (1, 100, 20, 17, 1), (2, 29, 24, 24, 2),
    (1, 37, 33, 33, 1), (2, 23, 70, 64, 1), (1, 300, 32, 16, 1), (1, 517, 16, 2, 1), (5, 9, 80, 16, 5),
    (1, 300, 16, 40, 1), (2, 210, 36, 24, 2), (1, 260, 48, 32, 1), (1, 145, 8, 4, 1)])
def test_sizes(gpu_device, batch, length, channels, states, groups, dtype):
    print(f"[case] scan {batch}x{length}x{channels}x{states} groups={groups} {dtype}", flush=True)
    _check(gpu_device, np.random.default_rng(length * 100 + states), batch, length, channels, states, groups, dtype)


@pytest.mark.parametrize("layout", ["plain", "window", "tokens"])
@pytest.mark.parametrize("use_softplus,without", [
    (True, ("z",)), (True, ("D", "delta_bias", "initial", "gfinal")), (False, ()), (False, ("z", "D", "initial"))])
def test_layouts_and_options(gpu_device, layout, use_softplus, without):
    print(f"[case] scan layout={layout} softplus={use_softplus} without={without}", flush=True)
    _check(gpu_device, np.random.default_rng(8), 3, 45, 40, 16, 2, "float32", use_softplus, without, layout)


@pytest.mark.parametrize("states,longest", [(16, 70), (6, 70), (24, 70), (16, 400), (33, 400), (8, 400)])
def test_packed(gpu_device, states, longest):
    """Empty, one-token and longer sequences that end inside a segment, rows
    that belong to none (NaN there reaches nothing; outputs stay as they were)."""
    import ferrum_gpu
    rng = np.random.default_rng(states)
    channels, groups = 24, 2
    lengths = [0, 1, longest - 1, 16, 0, 33, longest]
    offsets = np.concatenate([[3], 3 + np.cumsum(lengths)])
    tokens = int(offsets[-1]) + 4
    n = len(lengths)
    i = _inputs(rng, (tokens,), channels, states, groups, "float32", n)
    for k in ("u", "delta", "z", "B", "C", "gy"):
        i[k][:3] = i[k][offsets[-1]:] = float("nan")
    d = {k: up(v) for k, v in i.items()}
    got = {"out": fill(i["u"].shape), "final": fill(i["initial"].shape), "initial": fill(i["initial"].shape)}
    got.update({k: fill(i[k].shape) for k in GRADS})
    off = up(torch.from_numpy(offsets.astype(np.int32)))
    plan = ferrum_gpu.ssm.ScanPlan(n, longest, channels, states, gpu_device, groups=groups, dtype="float32",
                                   tokens=tokens)
    check = room(plan.checkpoint_bytes)
    opt = {k: d[k] for k in ("D", "z", "delta_bias")}
    main = [d[k] for k in ("u", "delta", "A", "B", "C")]
    plan.forward(*main, got["out"], **opt, initial=d["initial"], final=got["final"], offsets=off, checkpoints=check)
    plan.backward(*main, d["gy"], check, **opt, **{"grad_" + k: got[k] for k in GRADS}, grad_initial=got["initial"],
                  grad_final=d["gfinal"], offsets=off)
    gpu_device.sync()
    _compare(got, i, [((slice(int(offsets[s]), int(offsets[s + 1])),), s) for s in range(n)], channels, groups,
             states, "float32")
    for k in ("out", "u", "delta", "z", "B", "C"):
        assert (got[k][:3] == 7).all() and (got[k][offsets[-1]:] == 7).all(), k
    # offsets out of order or beyond the rows touch nothing outside them
    got["out"].fill_(7)
    off.copy_(torch.tensor([-4, 2, 9, 5, 2 ** 31 - 1, 1, 1, 1][:n + 1], dtype=torch.int32))
    plan.forward(*main, got["out"], **opt, initial=d["initial"], final=got["final"], offsets=off, checkpoints=check)
    plan.backward(*main, d["gy"], check, **opt, **{"grad_" + k: got[k] for k in GRADS}, offsets=off)
    gpu_device.sync()


def test_no_tokens(gpu_device):
    """No sequences, or sequences without tokens: states pass through, parameter gradients are zeros."""
    import ferrum_gpu
    for batch, length in ((0, 5), (2, 0)):
        i = {k: up(v) for k, v in _inputs(np.random.default_rng(0), (batch, length), 16, 8, 1, "float32",
                                             batch).items()}
        fin, gini, gA = fill((batch, 16, 8)), fill((batch, 16, 8)), fill((16, 8))
        plan = ferrum_gpu.ssm.ScanPlan(batch, length, 16, 8, gpu_device, dtype="float32")
        check = room(plan.checkpoint_bytes)
        main = [i[k] for k in ("u", "delta", "A", "B", "C")]
        plan.forward(*main, like(i["u"]), initial=i["initial"], final=fin, checkpoints=check)
        plan.backward(*main, i["gy"], check, grad_A=gA, grad_initial=gini, grad_final=i["gfinal"])
        gpu_device.sync()
        assert same(fin, i["initial"]) and same(gini, i["gfinal"]) and (gA == 0).all()


def test_rows_of_no_sequence(gpu_device):
    """Packed rows without any sequence: nothing is read or written, parameter gradients are zeros."""
    import ferrum_gpu
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(0), (9,), 16, 8, 1, "float32", 0).items()}
    off = up(torch.zeros(1, dtype=torch.int32))
    out, gB, gC, gA = fill((9, 16)), fill((9, 1, 8)), fill((9, 1, 8)), fill((16, 8))
    plan = ferrum_gpu.ssm.ScanPlan(0, 5, 16, 8, gpu_device, dtype="float32", tokens=9)
    check = room(plan.checkpoint_bytes)
    main = [i[k] for k in ("u", "delta", "A", "B", "C")]
    plan.forward(*main, out, offsets=off, checkpoints=check)
    plan.backward(*main, i["gy"], check, grad_A=gA, grad_B=gB, grad_C=gC, offsets=off)
    gpu_device.sync()
    assert all((v.get() == 7).all() for v in (out, gB, gC)) and (gA == 0).all()


@pytest.mark.parametrize("length", [5, 900])
def test_final_may_be_initial(gpu_device, length):
    """Also where the token axis is split: no part reads what another has written."""
    import ferrum_gpu
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(1), (1, length), 32, 16, 1, "float32", 1).items()}
    plan = ferrum_gpu.ssm.ScanPlan(1, length, 32, 16, gpu_device, dtype="float32")
    main = [i[k] for k in ("u", "delta", "A", "B", "C")]
    a, b, fin, state = like(i["u"]), like(i["u"]), fill((1, 32, 16)), i["initial"].clone()
    plan.forward(*main, a, initial=i["initial"], final=fin)
    plan.forward(*main, b, initial=state, final=state)
    gpu_device.sync()
    assert same(a, b) and same(fin, state)


def test_same_bits_again(gpu_device):
    """Sums over channels and tokens do not depend on timing."""
    import ferrum_gpu
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(4), (2, 333), 200, 16, 1, "bfloat16", 2).items()}
    plan = ferrum_gpu.ssm.ScanPlan(2, 333, 200, 16, gpu_device)
    check = room(plan.checkpoint_bytes)
    main, opt = [i[k] for k in ("u", "delta", "A", "B", "C")], {k: i[k] for k in ("D", "z", "delta_bias")}
    runs = []
    for _ in range(3):
        got = {k: like(i[k]) for k in GRADS}
        out = like(i["u"])
        plan.forward(*main, out, **opt, checkpoints=check)
        plan.backward(*main, i["gy"], check, **opt, **{"grad_" + k: v for k, v in got.items()})
        gpu_device.sync()
        runs.append([out, *got.values()])
    for other in runs[1:]:
        assert all(same(x, y) for x, y in zip(runs[0], other))


def test_gradient_is_the_difference(gpu_device):
    """Along a random direction of every input, the GPU's own forward pass (in
    float32, its loss summed in 64 bits) changes by what the gradient says.
    The step h = 2^-6 leaves the third derivative's h^2 / 6 and rounding of
    about 2^-24 * sqrt(values) / h of the loss's size; 2e-3 is over four times
    what both come to for these sizes."""
    import ferrum_gpu
    rng = np.random.default_rng(6)
    batch, length, channels, states = 2, 40, 24, 16
    i = {k: up(v) for k, v in _inputs(rng, (batch, length), channels, states, 1, "float32", batch).items()}
    plan = ferrum_gpu.ssm.ScanPlan(batch, length, channels, states, gpu_device, dtype="float32")
    check = room(plan.checkpoint_bytes)

    def loss(j):
        out, fin = like(j["u"]), like(j["initial"])
        plan.forward(*(j[k] for k in ("u", "delta", "A", "B", "C")), out, D=j["D"], z=j["z"],
                     delta_bias=j["delta_bias"], initial=j["initial"], final=fin, checkpoints=check)
        gpu_device.sync()
        return float((values(out) * values(i["gy"])).sum() + (values(fin) * values(i["gfinal"])).sum())

    loss(i)
    got = {k: like(i[k]) for k in GRADS + ("initial",)}
    plan.backward(*(i[k] for k in ("u", "delta", "A", "B", "C")), i["gy"], check, D=i["D"], z=i["z"],
                  delta_bias=i["delta_bias"], **{"grad_" + k: v for k, v in got.items()}, grad_final=i["gfinal"])
    gpu_device.sync()
    for k, g in got.items():
        v = torch.from_numpy(rng.standard_normal(tuple(g.shape))).float()
        v /= v.norm()
        h = 2.0 ** -6
        want = (loss({**i, k: up(i[k].get() + h * v)}) - loss({**i, k: up(i[k].get() - h * v)})) / (2 * h)
        g = g.get().double()
        assert abs((g * v).sum().item() - want) <= 2e-3 * g.norm().item(), k


@pytest.mark.parametrize("states", [16, 13, 6, 33])
def test_nothing_leaks(gpu_device, states):
    """A channel, a sequence and a later token that hold NaN or infinity leave
    all others as they are; an infinite time step forgets (its own channel
    only), whatever the number of states."""
    import ferrum_gpu
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(3), (2, 50), 40, states, 1, "float32", 2).items()}
    plan = ferrum_gpu.ssm.ScanPlan(2, 50, 40, states, gpu_device, dtype="float32")

    def run(j):
        out, fin = like(j["u"]), fill((2, 40, states))
        plan.forward(*(j[k] for k in ("u", "delta", "A", "B", "C")), out, D=j["D"], z=j["z"],
                     delta_bias=j["delta_bias"], initial=j["initial"], final=fin)
        gpu_device.sync()
        return out.get(), fin.get()

    good, good_fin = run(i)
    j = {k: v.clone() for k, v in i.items()}
    j["u"][0, 30, 5] = float("nan")
    j["z"][0, 20, 9] = float("inf")
    j["initial"][1, 7] = float("nan")
    j["B"][1, 49] = float("nan")
    out, fin = run(j)
    touched = torch.zeros_like(out, dtype=torch.bool)
    touched[0, 30:, 5] = touched[0, 20, 9] = touched[1, :, 7] = touched[1, 49] = True
    assert same(out[~touched], good[~touched])
    assert torch.isnan(out[0, 30:, 5]).all() and torch.isinf(out[0, 20, 9]) and torch.isnan(out[1, :, 7]).all()
    keep = [c for c in range(40) if c != 5]
    assert same(fin[0, keep], good_fin[0, keep])
    # delta = inf with u = 0 at a token: the decay is 0, the input inf * 0 = NaN
    # for this channel; delta = inf and u > 0: infinite states of B's signs
    k = {n: v.clone() for n, v in i.items()}
    k["delta"][0, 10, 3] = float("inf")
    k["u"][0, 10, 3] = 1.0
    out, fin = run(k)
    b = i["B"].get()[0, 10, 0]
    assert torch.isinf(fin[0, 3]).all() and same(fin[0, 3] > 0, b > 0)
    keep = [c for c in range(40) if c != 3]
    assert same(out[0][:, keep], good[0][:, keep]) and same(out[1], good[1])
    # A = -inf: such a state holds only its own token's input
    m = {n: v.clone() for n, v in i.items()}
    m["A"][11] = float("-inf")
    out, fin = run(m)
    raw = values((i["delta"].get() + i["delta_bias"].get())[:, -1, 11])
    want = (o.softplus(raw) * values(i["u"][:, -1, 11]))[:, None] * values(i["B"][:, -1, 0])
    assert np.allclose(values(fin[:, 11]), want, rtol=1e-5, atol=1e-30)


@pytest.mark.parametrize("length", [30, 700])
def test_a_constant_scan_is_the_ffts_filter(gpu_device, length):
    """With a constant time step, B and C the scan is the convolution with
    k_t = sum_n C_n exp(t dt A_n) dt B_n, which the package's FFT computes:
    transform, product, normalised inverse, of padded signals.  Bound: the FFT's
    1e-4 relative to the largest value."""
    import ferrum_gpu
    from ferrum_gpu import pointwise
    rng = np.random.default_rng(12)
    channels, states = 8, 16
    i = _inputs(rng, (1, length), channels, states, 1, "float32", 1)
    i["delta"].zero_()
    i["B"][:], i["C"][:] = i["B"][:, :1].clone(), i["C"][:, :1].clone()
    u = i["u"][0].t()
    i = {k: up(v) for k, v in i.items()}
    out = like(i["u"])
    plan = ferrum_gpu.ssm.ScanPlan(1, length, channels, states, gpu_device, dtype="float32")
    plan.forward(*(i[k] for k in ("u", "delta", "A", "B", "C")), out, delta_bias=i["delta_bias"])
    log_n = (2 * length - 1).bit_length()
    dt = o.softplus(values(i["delta_bias"]))
    t = np.arange(length)
    kernel = np.einsum("n,tdn,n,d->dt", values(i["C"])[0, 0, 0], np.exp(t[:, None, None] * dt[:, None] * values(i["A"])),
                       values(i["B"])[0, 0, 0], dt)
    both = torch.zeros(2, channels, 1 << log_n, dtype=torch.complex64)
    both[0, :, :length], both[1, :, :length] = u, torch.from_numpy(kernel)
    both = up(both)
    fft, back = (ferrum_gpu.fft.Plan1D(log_n, n, gpu_device) for n in (2 * channels, channels))
    fft.execute(both, both, "forward")
    pointwise.cmul(gpu_device, both[0], both[1], both[0], channels << log_n)
    back.execute(both[0], both[0], "inverse", normalize=True)
    gpu_device.sync()
    want = both.get()[0, :, :length].real.t()
    assert (out.get()[0] - want).abs().max().item() <= 1e-4 * want.abs().max().item()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("batch,channels,states,groups", [(1, 16, 16, 1), (4, 70, 16, 2), (3, 33, 1, 1), (2, 30, 5, 3),
                                                          (5, 64, 13, 1), (2, 24, 33, 2), (3, 1000, 64, 1)])
def test_step(gpu_device, batch, channels, states, groups, dtype):
    """Slots in any order, one row without a slot and one beyond the states;
    the states of no row stay as they are."""
    import ferrum_gpu
    rng = np.random.default_rng(batch * 100 + states)
    rows = batch + 2
    i = _inputs(rng, (batch,), channels, states, groups, dtype, rows)
    st = i["initial"]
    slots = rng.permutation(rows)[:batch].astype(np.int32)
    if batch > 2:
        slots[0], slots[1] = -1, rows
    d = {k: up(v) for k, v in i.items()}
    for in_place, without in ((True, ()), (False, ("z", "D", "delta_bias"))):
        state, out = up(st), fill((batch, channels), dtype)
        new = None if in_place else state.clone()
        opt = {k: d[k] for k in ("D", "z", "delta_bias") if k not in without}
        ds = up(torch.from_numpy(slots))
        ferrum_gpu.ssm.scan_step(gpu_device, d["u"], d["delta"], d["A"], d["B"], d["C"], state, out, slots=ds,
                                 state_out=new, **opt)
        gpu_device.sync()
        after = state if in_place else new
        free = np.ones(rows, bool)
        for r, s in enumerate(slots):
            if s < 0 or s >= rows:
                assert (out[r] == 0).all()
                continue
            free[s] = False
            a = _oracle_args({**i, "initial": st[int(s)][None].expand(batch, -1, -1)}, slice(r, r + 1), r, True,
                             without + ("gfinal",))
            want, m = o.scan(**a), o.scan(**a, magnitude=True)
            rounds = o.scan_rounds(1, a["A"], 5.0, states)
            o.within(values(out[r]), want["out"][0], m["out"][0], rounds, dtype, "out")
            o.within(values(after[int(s)]), want["final"], m["final"], rounds, "float32", "state")
        assert same(after.get()[torch.from_numpy(free)], st[torch.from_numpy(free)])
        if not in_place:
            assert same(state, st)


def test_step_many_rows(gpu_device):
    """Rows enough for a wave to walk through several, the last wave fewer."""
    import ferrum_gpu
    rng = np.random.default_rng(21)
    batch, channels, states = 33001, 16, 16
    i = _inputs(rng, (batch,), channels, states, 1, "float32", batch)
    d = {k: up(v) for k, v in i.items()}
    out, slots = fill((batch, channels)), up(torch.from_numpy(rng.permutation(batch).astype(np.int32)))
    slots[5], slots[batch - 1] = -1, batch
    state = d["initial"].clone()
    ferrum_gpu.ssm.scan_step(gpu_device, d["u"], d["delta"], d["A"], d["B"], d["C"], state, out, D=d["D"], z=d["z"],
                             delta_bias=d["delta_bias"], slots=slots)
    gpu_device.sync()
    n = {k: values(v) for k, v in i.items()}
    s = slots.get().numpy()
    on = (s >= 0) & (s < batch)
    dt = o.softplus(n["delta"] + n["delta_bias"])
    a = np.exp(dt[:, :, None] * n["A"])
    prior = n["initial"][np.where(on, s, 0)]
    want, m = ((f(a * prior) if f is np.abs else a * prior) + f((dt * n["u"])[:, :, None] * n["B"][:, 0][:, None])
               for f in (lambda v: v, np.abs))
    rounds = o.scan_rounds(1, n["A"], float(dt.max()), states)
    after = values(state)
    o.within(after[s[on]], want[on], m[on], rounds, "float32", "state")
    untouched = np.ones(batch, bool)
    untouched[s[on]] = False
    assert np.array_equal(after[untouched], n["initial"][untouched])
    gate = n["z"] * o.sigmoid(n["z"])
    y = ((want * n["C"][:, 0][:, None]).sum(-1) + n["D"] * n["u"]) * gate
    my = ((m * np.abs(n["C"][:, 0][:, None])).sum(-1) + np.abs(n["D"] * n["u"])) * np.abs(gate)
    o.within(values(out)[on], y[on], my[on], rounds, "float32", "out")
    assert (values(out)[~on] == 0).all()


def test_windows_of_one_array(gpu_device):
    """One token of each row: inputs and outputs that are columns of one array."""
    import ferrum_gpu
    d, n = 32, 16
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(2), (3, 1), d, n, 1, "float32", 3).items()}
    big = up(torch.zeros(3, 1, 4 * d + 2 * n))
    big[..., :d], big[..., d:2 * d], big[..., 2 * d:3 * d] = i["u"], i["delta"], i["z"]
    big[..., 4 * d:4 * d + n], big[..., 4 * d + n:] = i["B"][:, :, 0], i["C"][:, :, 0]
    plan = ferrum_gpu.ssm.ScanPlan(3, 1, d, n, gpu_device, dtype="float32")
    want, state = like(i["u"]), i["initial"].clone()
    cols = [big[..., k * d:(k + 1) * d] for k in range(4)]
    b, c = big[..., 4 * d:4 * d + n], big[..., 4 * d + n:]
    plan.forward(i["u"], i["delta"], i["A"], i["B"], i["C"], want, z=i["z"], initial=i["initial"])
    plan.forward(cols[0], cols[1], i["A"], b, c, cols[3], z=cols[2], initial=i["initial"])
    gpu_device.sync()
    assert same(cols[3], want)
    cols[3].fill_(0)
    ferrum_gpu.ssm.scan_step(gpu_device, cols[0][:, 0], cols[1][:, 0], i["A"], b[:, 0], c[:, 0], state, cols[3][:, 0],
                             z=cols[2][:, 0])
    gpu_device.sync()
    assert torch.allclose(cols[3].get(), want.get(), rtol=1e-5, atol=1e-5)


def test_prompt_then_tokens(gpu_device):
    """A prompt and single tokens after it are the whole sequence, within what
    32 bits leave."""
    import ferrum_gpu
    ssm = ferrum_gpu.ssm
    batch, length, more, channels, states = 2, 21, 6, 48, 16
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(7), (batch, length + more), channels, states, 1,
                                         "float32", batch).items()}
    rows, opt = ("u", "delta", "B", "C", "z"), {k: i[k] for k in ("D", "delta_bias")}
    whole, out, state, fin = like(i["u"]), like(i["u"]), i["initial"].clone(), \
        like(i["initial"])

    def forward(n, to, **k):
        r = {x: i[x][:, :n] for x in rows}
        ssm.ScanPlan(batch, n, channels, states, gpu_device, dtype="float32").forward(
            r["u"], r["delta"], i["A"], r["B"], r["C"], to[:, :n], z=r["z"], **opt, **k)
        gpu_device.sync()  # the plan's workspace is freed here

    forward(length + more, whole, initial=i["initial"], final=fin)
    forward(length, out, initial=state, final=state)
    for t in range(length, length + more):
        r = {x: i[x][:, t] for x in rows}
        ssm.scan_step(gpu_device, r["u"], r["delta"], i["A"], r["B"], r["C"], state, out[:, t], z=r["z"], **opt)
    gpu_device.sync()
    assert all(torch.allclose(x.get(), y.get(), rtol=1e-5, atol=1e-5) for x, y in ((out, whole), (state, fin)))


def test_broadcast_inputs(gpu_device):
    """B and C that all sequences share (stride 0): read as they are; their
    gradients come for each sequence."""
    import ferrum_gpu
    batch, length, channels, states = 3, 20, 32, 16
    i = _inputs(np.random.default_rng(8), (batch, length), channels, states, 1, "float32", batch)
    for k in ("B", "C"):
        i[k] = i[k][:1].expand(batch, -1, -1, -1)
    d = {k: up(v) for k, v in i.items()}
    assert d["B"].stride()[0] == 0
    plan = ferrum_gpu.ssm.ScanPlan(batch, length, channels, states, gpu_device, dtype="float32")
    check = room(plan.checkpoint_bytes)
    got = {k: fill(i[k].shape) for k in GRADS}
    got["out"] = fill(i["u"].shape)
    main, opt = [d[k] for k in ("u", "delta", "A", "B", "C")], {k: d[k] for k in ("D", "z", "delta_bias")}
    plan.forward(*main, got["out"], **opt, checkpoints=check)
    plan.backward(*main, d["gy"], check, **opt, **{"grad_" + k: got[k] for k in GRADS})
    gpu_device.sync()
    _compare(got, i, [((s, slice(0, length)), s) for s in range(batch)], channels, 1, states, "float32",
             without=("initial", "gfinal"))


def test_another_stream_and_captured_calls(gpu_device):
    """On a stream of the caller's, and in a graph replayed with other inputs."""
    import ferrum_gpu
    from ferrum_gpu.hip import Capture, Stream
    from ferrum_gpu._native import FerrumGpuError
    ssm = ferrum_gpu.ssm
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(9), (1, 600), 64, 16, 1, "float32", 1).items()}
    plan = ssm.ScanPlan(1, 600, 64, 16, gpu_device, dtype="float32")
    check = room(plan.checkpoint_bytes)
    got = {k: like(i[k]) for k in GRADS}
    out, so, new = like(i["u"]), fill((1, 64)), fill((1, 64, 16))
    main, opt = [i[k] for k in ("u", "delta", "A", "B", "C")], {k: i[k] for k in ("D", "z", "delta_bias")}

    def calls(stream):
        plan.forward(*main, out, **opt, initial=i["initial"], checkpoints=check, stream=stream)
        plan.backward(*main, i["gy"], check, **opt, **{"grad_" + k: v for k, v in got.items()}, stream=stream)
        ssm.scan_step(gpu_device, i["u"][:, 0], i["delta"][:, 0], i["A"], i["B"][:, 0], i["C"][:, 0], i["initial"],
                      so, state_out=new, stream=stream)

    every = [out, so, new, *got.values()]
    with pytest.raises(FerrumGpuError, match="cannot be captured"):
        with Capture(gpu_device) as cap:
            calls(cap.stream)
    calls(0)
    stream = Stream(gpu_device)
    with Capture(gpu_device, keep=[plan]) as cap:
        calls(cap.stream)
    for k in range(4):
        for n in ("u", "delta", "gy", "B", "C"):
            i[n].normal_()
        calls(0)
        gpu_device.sync()
        want = [v.clone() for v in every]
        for run in (lambda: calls(stream.handle), cap.graph.launch):
            for v in every:
                v.fill_(7)
            run()
            stream.sync()
            gpu_device.sync()
            assert all(same(a, b) for a, b in zip(want, every)), k


def test_rows_far_apart(gpu_device):
    """Rows whose distance from the first passes 2^32 bytes."""
    import ferrum_gpu
    from ferrum_gpu.hip import DeviceBuffer
    row, length = 1 << 25, 70
    host = _inputs(np.random.default_rng(5), (1, length), 64, 16, 1, "float16", 1)
    i = {k: up(v) for k, v in host.items()}
    big = DeviceBuffer(gpu_device, 2 * length * row)
    f = {**i, **{k: Far(big, host[k], row, 100 * at) for at, k in enumerate(("u", "delta", "z", "B", "C"))}}
    plan = ferrum_gpu.ssm.ScanPlan(1, length, 64, 16, gpu_device, dtype="float16")
    outs = [like(i["u"]), Far(big, torch.zeros(1, length, 64, dtype=torch.float16), row, 1000)]
    for j, out in zip((i, f), outs):
        plan.forward(*(j[k] for k in ("u", "delta", "A", "B", "C")), out, z=j["z"])
    gpu_device.sync()
    assert same(*outs)


def test_refusals(gpu_device):
    import ferrum_gpu
    from ferrum_gpu import _native as N
    ssm, E = ferrum_gpu.ssm, N.FerrumGpuError
    make = lambda **k: ssm.ScanPlan(**{**dict(batch=2, length=8, channels=16, states=4, device=gpu_device,  # noqa: E731
                                              groups=2, dtype="float32"), **k})
    for bad in (dict(states=0), dict(states=65), dict(channels=0), dict(groups=0), dict(batch=-1), dict(length=-2),
                dict(groups=17)):
        with pytest.raises(E, match="must be in"):
            make(**bad)
    with pytest.raises(E, match="groups must divide"):
        make(groups=3)
    for bad in (dict(channels=(1 << 25) + 8), dict(channels=1 << 25, groups=1 << 24)):
        with pytest.raises(E, match="must be in"):
            make(length=1, batch=1, **bad)
    with pytest.raises(E, match="too large"):
        make(batch=(1 << 31) - 1, length=1, channels=1 << 25, groups=1)
    plan = make()
    x, out = up(torch.zeros(2, 8, 16)), up(torch.zeros(2, 8, 16))
    A, D = up(torch.zeros(16, 4)), up(torch.zeros(16))
    B, C = up(torch.zeros(2, 8, 2, 4)), up(torch.zeros(2, 8, 8))
    st = up(torch.zeros(2, 16, 4))
    check = room(plan.checkpoint_bytes)
    delta = like(x)
    plan.forward(x, delta, A, B, C, out, checkpoints=check)
    with pytest.raises(ValueError, match="shape"):
        plan.forward(x, delta, up(A.get().t().contiguous()), B, C, out)
    with pytest.raises(ValueError, match="shape"):
        plan.forward(x, delta, A, B[..., :3], C, out)
    with pytest.raises(ValueError, match="bfloat16"):
        plan.forward(up(x.get().bfloat16()), delta, A, B, C, out)
    with pytest.raises(ValueError, match="float64"):
        plan.forward(x, delta, A, B, C, out, D=up(D.get().double()))
    with pytest.raises(ValueError, match="runs on GPU"):
        plan.forward(x, delta, A.get(), B, C, out)
    with pytest.raises(ValueError, match="checkpoints"):
        plan.forward(x, delta, A, B, C, out, checkpoints=check[:-1])
    with pytest.raises(ValueError, match="shape"):
        plan.forward(x, delta, A, B, C, out, initial=st[:1])
    with pytest.raises(E, match="null buffer"):
        plan.forward(x, None, A, B, C, out)
    with pytest.raises(E, match="null buffer"):
        plan.backward(x, delta, A, B, C, out, None)
    with pytest.raises(E, match="overlap"):
        plan.forward(x, delta, A, B, C, x)
    with pytest.raises(E, match="overlap"):
        plan.forward(x, delta, A, B, C, out, final=out.view(-1)[:128].view(2, 16, 4))
    with pytest.raises(E, match="overlap"):
        plan.backward(x, delta, A, B, C, out, check, grad_u=delta)
    with pytest.raises(E, match="grad_z without z"):
        plan.backward(x, delta, A, B, C, out, check, grad_z=like(x))
    with pytest.raises(ValueError, match="only packed"):
        plan.forward(x, delta, A, B, C, out, offsets=up(torch.zeros(3, dtype=torch.int32)))
    with pytest.raises(ValueError, match="int32"):
        make(tokens=16).forward(x.view(16, 16), delta.view(16, 16), A, B.view(16, 2, 4), C.view(16, 8),
                                out.view(16, 16), offsets=up(torch.zeros(3, dtype=torch.int64)))
    with pytest.raises(E, match="state_rows"):
        ssm.scan_step(gpu_device, x[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], st[:1], out[:, 0])
    with pytest.raises(ValueError, match="slots"):
        ssm.scan_step(gpu_device, x[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], st, out[:, 0],
                      slots=up(torch.zeros(3, dtype=torch.int32)))
    with pytest.raises(ValueError, match="B: shape"):
        ssm.scan_step(gpu_device, x[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], st, out[:, 0], groups=0)
    plan.destroy()
    with pytest.raises(ValueError, match="destroyed"):
        plan.forward(x, delta, A, B, C, out)
    gpu_device.sync()


@pytest.mark.parametrize("states", [16, 5])
def test_parts_of_growing_and_shrinking_states(gpu_device, states):
    """States that are 0, or so small or large, that they stay finite token by
    token, under factors of a part of the tokens (here e^96 and e^-96) that
    32 bits do not hold; forward and backward."""
    import ferrum_gpu
    length, channels = 300, 16
    i = _inputs(np.random.default_rng(13), (1, length), channels, states, 1, "float32", 1)
    i["A"].fill_(3.0)
    i["delta"].fill_(1.0)
    i["delta_bias"].zero_()
    # channels 0 .. 7: nothing comes in before the last tokens, no gradient after the first
    i["u"][:, :-5] = i["gy"][:, 5:] = 0
    i["initial"][:, :8] = i["gfinal"][:, :8] = 0
    # the others: 32 tokens up, 32 down, four times; or down, then up
    turns = torch.arange(length) // 32 % 2 == 1
    i["delta"][0, turns, 8:] = -1
    i["delta"][0, 256:, 8:] = 0
    i["delta"][:, :, 12:] *= -1
    i["initial"][:, 8:12], i["initial"][:, 12:] = 1e-30, 1e30
    i["gfinal"][:, 8:12], i["gfinal"][:, 12:] = 1e30, 1e-30
    i["u"][:, :, 8:] = i["gy"][:, :, 8:] = 0
    d = {k: up(v) for k, v in i.items()}
    plan = ferrum_gpu.ssm.ScanPlan(1, length, channels, states, gpu_device, dtype="float32", softplus=False)
    check = room(plan.checkpoint_bytes)
    got = {"out": fill(i["u"].shape), "final": fill(i["initial"].shape), "initial": fill(i["initial"].shape)}
    grads = ("u", "delta", "A")
    got.update({k: fill(i[k].shape) for k in grads})
    main = [d[k] for k in ("u", "delta", "A", "B", "C")]
    plan.forward(*main, got["out"], initial=d["initial"], final=got["final"], checkpoints=check)
    plan.backward(*main, d["gy"], check, **{"grad_" + k: got[k] for k in grads}, grad_initial=got["initial"],
                  grad_final=d["gfinal"])
    gpu_device.sync()
    a = _oracle_args(i, (0, slice(0, length)), 0, False, ("z", "D"))
    r, m = o.scan(**a), o.scan(**a, magnitude=True)
    # as _compare(), with a sum of the time steps and its product in each of ten parts
    rounds = o.scan_rounds(length, a["A"], 1.0, states) + 10 * (34 + 3 * 32)
    o.within(values(got["out"][0]), r["out"], m["out"], rounds, "float32", "out")
    o.within(values(got["final"][0]), r["final"], m["final"], rounds, "float32", "final")
    o.within(values(got["initial"][0]), r["initial"], m["initial"], rounds, "float32", "grad_initial")
    for k in ("u", "delta"):
        o.within(values(got[k][0]), r[k], m[k], 2 * rounds, "float32", "grad_" + k)
    o.within(values(got["A"]), r["A"], m["A"], 2 * rounds + length, "float32", "grad_A")
    assert (values(got["final"])[0, 8:] != 0).all() and (values(got["initial"])[0, 8:] != 0).all()


@pytest.mark.parametrize("longest", [1000, 21])
@pytest.mark.parametrize("states", [16, 24])
def test_packed_parameter_gradients(gpu_device, states, longest):
    """Many short sequences and a plan for much longer ones, or for shorter
    ones (which cuts them): nothing of an earlier call's other sequences, rows
    before, between or after is in the sums."""
    import ferrum_gpu
    rng = np.random.default_rng(17 + states)
    tokens, channels, n = 700, 24, 30
    i = _inputs(rng, (tokens,), channels, states, 1, "float32", n)
    d = {k: up(v) for k, v in i.items()}
    plan = ferrum_gpu.ssm.ScanPlan(n, longest, channels, states, gpu_device, dtype="float32", tokens=tokens)
    assert plan.describe()["backward_parts"] > (10 if longest == 1000 else 0)
    check = room(plan.checkpoint_bytes)
    opt = {k: d[k] for k in ("D", "z", "delta_bias")}
    main = [d[k] for k in ("u", "delta", "A", "B", "C")]
    for start, most in ((0, 46), (17, 30), (300, 3)):
        lengths = rng.integers(0, most, n)
        offsets = np.minimum(start + np.concatenate([[0], np.cumsum(lengths)]), tokens)
        off = up(torch.from_numpy(offsets.astype(np.int32)))
        got = {"out": fill(i["u"].shape), "final": fill(i["initial"].shape), "initial": fill(i["initial"].shape)}
        got.update({k: fill(i[k].shape) for k in GRADS})
        plan.forward(*main, got["out"], **opt, initial=d["initial"], final=got["final"], offsets=off,
                     checkpoints=check)
        plan.backward(*main, d["gy"], check, **opt, **{"grad_" + k: got[k] for k in GRADS},
                      grad_initial=got["initial"], grad_final=d["gfinal"], offsets=off)
        gpu_device.sync()
        spans = [((slice(int(a), int(min(b, a + longest))),), s) for s, (a, b) in enumerate(zip(offsets, offsets[1:]))]
        _compare(got, i, spans, channels, 1, states, "float32")


def test_workspaces_go_by_rows(gpu_device):
    """Packed: not by as many tokens for every sequence as the longest has, and
    the backward pass's from its first call on."""
    import ferrum_gpu
    n, longest, tokens, channels, states = 1024, 4096, 4096, 64, 16
    plan = ferrum_gpu.ssm.ScanPlan(n, longest, channels, states, gpu_device, dtype="float32", tokens=tokens)
    before = plan.describe()
    assert before["forward_parts"] > 10
    # a state of each channel, and its time step, for every part; a state for each sequence's initial ones
    parts = tokens // before["forward_tokens"] + n
    assert before["workspace_bytes"] == 4 * channels * (states * (parts + n) + parts)
    i = {k: up(v) for k, v in _inputs(np.random.default_rng(0), (tokens,), channels, states, 1, "float32", 0).items()}
    off = up(torch.arange(0, tokens + 1, 4, dtype=torch.int32))
    check, gA = room(plan.checkpoint_bytes), fill((channels, states))
    main = [i[k] for k in ("u", "delta", "A", "B", "C")]
    plan.forward(*main, like(i["u"]), offsets=off, checkpoints=check)
    plan.backward(*main, i["gy"], check, grad_A=gA, offsets=off)
    gpu_device.sync()
    after, parts = plan.describe(), tokens // before["backward_tokens"] + n
    assert after["workspace_bytes"] - before["workspace_bytes"] == \
        4 * channels * (states * (parts + n) + parts) + 4 * channels * (states + 2) * parts + 4 * tokens * 2 * states
    one = ferrum_gpu.ssm.ScanPlan(64, 100, 512, states, gpu_device, dtype="float32")
    assert one.describe()["forward_parts"] == 1 and one.describe()["workspace_bytes"] == 0


def test_gradients_of_offsets_beyond_the_rows(gpu_device):
    """Offsets before the first row or behind the last are taken as those, by
    every gradient alike; the sequences are cut at the plan's length."""
    import ferrum_gpu
    rng = np.random.default_rng(19)
    tokens, channels, states, longest = 60, 24, 16, 33
    i = _inputs(rng, (tokens,), channels, states, 1, "float32", 3)
    d = {k: up(v) for k, v in i.items()}
    plan = ferrum_gpu.ssm.ScanPlan(3, longest, channels, states, gpu_device, dtype="float32", tokens=tokens)
    check = room(plan.checkpoint_bytes)
    main = [d[k] for k in ("u", "delta", "A", "B", "C")]
    for beyond, nearest in (([-5, 33, 40, 90], [0, 33, 40, 60]), ([-9, -3, 50, 70], [0, 0, 50, 60])):
        runs = []
        for offsets in (beyond, nearest):
            off = up(torch.tensor(offsets, dtype=torch.int32))
            got = [fill(i[k].shape) for k in ("u", "u", "A", "B", "C")]
            plan.forward(*main, got[0], offsets=off, checkpoints=check)
            plan.backward(*main, d["gy"], check, grad_u=got[1], grad_A=got[2], grad_B=got[3], grad_C=got[4],
                          offsets=off)
            gpu_device.sync()
            runs.append(got)
        assert all(same(a, b) for a, b in zip(*runs))
        rows = torch.zeros(tokens, dtype=torch.bool)
        for a, b in zip(nearest, nearest[1:]):
            rows[a:min(b, a + longest)] = True
        for g in runs[0][3:]:
            assert (g.get()[rows] != 7).all() and (g.get()[~rows] == 7).all()
