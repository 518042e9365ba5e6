"""The sequence filters on the GPU where their loops run longest: parts of the
token axis of many segments, long runs, packed sequences of every type, and NaN in
one place of an input.  Which parts and runs a plan has is asked of the plan, so
that a test does not pass for being cut differently."""

from __future__ import annotations

import numpy as np
import pytest

import ssm_oracle as o

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import gpu_tensor  # noqa: E402
from gpu_tensor import fill, like, room, same, up, values  # noqa: E402
from test_gpu_ssm_conv import _rounded, _rounds  # noqa: E402
from test_gpu_ssm_scan import GRADS, _compare, _inputs  # noqa: E402

SEGMENT = 16  # tokens that the scan works through at a time
MAIN = ("u", "delta", "A", "B", "C")


@pytest.fixture(autouse=True)
def _on_gpu(gpu_device):
    yield from gpu_tensor.use(gpu_device)


def _scan(dev, rng, lead, lengths, longest, channels, states, groups, dtype, least):
    """Forward and backward against the oracle; lengths: packed sequences, from
    row 3 on, NaN in the rows of none."""
    import ferrum_gpu
    batch = len(lengths) if lengths else lead[0]
    i = _inputs(rng, lead, channels, states, groups, dtype, batch)
    offsets = 3 + np.concatenate([[0], np.cumsum(lengths)]) if lengths else None
    off = {}
    if lengths:
        for k in ("u", "delta", "z", "B", "C", "gy"):
            i[k][:3] = i[k][offsets[-1]:] = float("nan")
        off["offsets"] = up(torch.from_numpy(offsets.astype(np.int32)))
    d = {k: up(v) for k, v in i.items()}
    got = {"out": fill(i["u"].shape, dtype), "final": fill(i["initial"].shape), "initial": fill(i["initial"].shape)}
    got.update({k: fill(i[k].shape, dtype if k in ("u", "delta", "z", "B", "C") else "float32") for k in GRADS})
    plan = ferrum_gpu.ssm.ScanPlan(batch, longest, channels, states, dev, groups=groups, dtype=dtype,
                                   tokens=lead[0] if lengths else None)
    parts = plan.describe()
    assert min(longest, parts["forward_tokens"]) // SEGMENT >= least[0], parts
    assert min(longest, parts["backward_tokens"]) // SEGMENT >= least[1], parts
    check = room(plan.checkpoint_bytes)
    opt = {k: d[k] for k in ("D", "z", "delta_bias")}
    main = [d[k] for k in MAIN]
    plan.forward(*main, got["out"], **opt, initial=d["initial"], final=got["final"], checkpoints=check, **off)
    plan.backward(*main, d["gy"], check, **opt, **{"grad_" + k: got[k] for k in GRADS}, grad_initial=got["initial"],
                  grad_final=d["gfinal"], **off)
    dev.sync()
    if not lengths:
        spans = [((s, slice(0, lead[1])), s) for s in range(batch)]
    else:
        spans = [((slice(int(a), int(b)),), s) for s, (a, b) in enumerate(zip(offsets, offsets[1:]))]
        for k in ("out", "u", "delta", "z", "B", "C"):
            assert (got[k].get()[:3] == 7).all() and (got[k].get()[offsets[-1]:] == 7).all(), k
    _compare(got, i, spans, channels, groups, states, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("full", range(3, 10))
def test_scan_parts_of_so_many_segments(gpu_device, full, dtype):
    """Whole segments and one that is not, vector accesses and any; groups
    enough that the axis is not cut."""
    for channels, length in ((2048, full * SEGMENT), (512, full * SEGMENT + 5)):
        print(f"[case] scan 1x{length}x{channels}x4 groups=512 {dtype}", flush=True)
        _scan(gpu_device, np.random.default_rng(full), (1, length), None, length, channels, 4, 512, dtype, (full, full))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("channels,states,groups", [
    (2048, 8, 512), (512, 6, 512), (2048, 16, 512), (512, 13, 512), (1024, 32, 512), (512, 24, 512), (256, 64, 256),
    (512, 40, 256)])
def test_scan_long_parts(gpu_device, channels, states, groups, dtype):
    """Every number of states and waves of a channel."""
    print(f"[case] scan 1x109x{channels}x{states} groups={groups} {dtype}", flush=True)
    _scan(gpu_device, np.random.default_rng(states), (1, 109), None, 109, channels, states, groups, dtype, (6, 6))


@pytest.mark.parametrize("dtype,length,channels,states", [
    ("bfloat16", 5127, 64, 16), ("float32", 5127, 48, 13), ("float16", 8500, 20, 8), ("bfloat16", 5200, 32, 33)])
def test_scan_long_sequence(gpu_device, dtype, length, channels, states):
    """One sequence, cut into parts of several segments, the last one shorter."""
    print(f"[case] scan 1x{length}x{channels}x{states} {dtype}", flush=True)
    _scan(gpu_device, np.random.default_rng(length), (1, length), None, length, channels, states, 1, dtype, (5, 5))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("channels,states,groups,longest", [
    (24, 16, 2, 70), (24, 6, 2, 400), (40, 8, 1, 400), (24, 24, 2, 400), (30, 33, 1, 70), (64, 64, 1, 70),
    (32, 32, 1, 400)])
def test_scan_packed_16_bits(gpu_device, channels, states, groups, longest, dtype):
    print(f"[case] scan packed {channels}x{states} groups={groups} longest={longest} {dtype}", flush=True)
    lengths = [0, 1, longest - 1, 16, 0, 33, longest]
    _scan(gpu_device, np.random.default_rng(states), (sum(lengths) + 7,), lengths, longest, channels, states, groups,
          dtype, (0, 0))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("channels,states,groups", [(2048, 16, 512), (512, 13, 512), (512, 24, 512), (256, 64, 256)])
def test_scan_packed_long_parts(gpu_device, channels, states, groups, dtype):
    print(f"[case] scan packed {channels}x{states} groups={groups} {dtype}", flush=True)
    lengths = [127, 0, 5, 128, 64]
    _scan(gpu_device, np.random.default_rng(states), (sum(lengths) + 7,), lengths, 128, channels, states, groups, dtype,
          (8, 8))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("width", [2, 4, 5, 8])
@pytest.mark.parametrize("channels", [40, 36, 37])
def test_conv_packed_16_bits(gpu_device, channels, width, dtype):
    """Empty, one-token and longer sequences, rows of none around them (NaN
    there reaches nothing; outputs stay as they were)."""
    import ferrum_gpu
    print(f"[case] conv packed {channels} width={width} {dtype}", flush=True)
    rng = np.random.default_rng(channels + width)
    lengths = [0, 1, 33, 0, 2, 29]
    offsets = 2 + np.concatenate([[0], np.cumsum(lengths)])
    tokens, n = int(offsets[-1]) + 3, len(lengths)
    x, gy = (_rounded(rng, (tokens, channels), dtype) for _ in range(2))
    for v in (x, gy):
        v[:2] = v[offsets[-1]:] = float("nan")
    w, b = (torch.from_numpy(rng.standard_normal(s)).float() for s in ((channels, width), (channels,)))
    ini, gf = (_rounded(rng, (n, width - 1, channels), dtype) for _ in range(2))
    out, gx, fin, gini = fill(x.shape, dtype), fill(x.shape, dtype), fill(ini.shape, dtype), fill(ini.shape, dtype)
    gw, gb = fill(w.shape), fill(b.shape)
    dx, dgy, dw, db, dini, dgf = (up(v) for v in (x, gy, w, b, ini, gf))
    off = up(torch.from_numpy(offsets.astype(np.int32)))
    plan = ferrum_gpu.ssm.ConvPlan(n, 33, channels, width, gpu_device, dtype=dtype, tokens=tokens)
    plan.forward(dx, dw, out, bias=db, initial=dini, final=fin, offsets=off)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw, grad_bias=gb, bias=db, initial=dini, grad_initial=gini,
                  grad_final=dgf, offsets=off)
    gpu_device.sync()
    want, size = [0, 0], [0, 0]
    for s, (i, j) in enumerate(zip(offsets, offsets[1:])):
        args = dict(x=values(x[i:j]), w=values(w), bias=values(b), initial=values(ini[s]), grad=values(gy[i:j]),
                    grad_final=values(gf[s]))
        r, m = o.conv(**args), o.conv(**args, magnitude=True)
        o.within(values(out[int(i):int(j)]), r["out"], m["out"], _rounds(width), dtype, "out")
        o.within(values(gx[int(i):int(j)]), r["x"], m["x"], _rounds(width), dtype, "grad_x")
        o.within(values(gini[s]), r["initial"], m["initial"], _rounds(width), dtype, "grad_initial")
        assert np.array_equal(values(fin[s]), r["final"])
        want, size = ([a[0] + v["weight"], a[1] + v["bias"]] for a, v in ((want, r), (size, m)))
    o.within(values(gw), want[0], size[0], _rounds(width, tokens), "float32", "grad_weight")
    o.within(values(gb), want[1], size[1], _rounds(width, tokens), "float32", "grad_bias")
    assert all((v.get()[:2] == 7).all() and (v.get()[offsets[-1]:] == 7).all() for v in (out, gx))


@pytest.mark.parametrize("dtype,width", [("bfloat16", 4), ("float16", 4), ("bfloat16", 2), ("float16", 8)])
def test_conv_long_runs(gpu_device, dtype, width):
    """Eight channels of a thread (up to four taps), runs of several groups of rows."""
    import ferrum_gpu
    print(f"[case] conv 1x140001x8 width={width} {dtype}", flush=True)
    rng = np.random.default_rng(width)
    length, channels = 140001, 8
    x, gy = (_rounded(rng, (1, length, channels), dtype) for _ in range(2))
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    plan = ferrum_gpu.ssm.ConvPlan(1, length, channels, width, gpu_device, dtype=dtype)
    runs = plan.describe()
    assert runs["forward_tokens"] >= 16 and runs["backward_tokens"] >= 16, runs
    out, gx, gw, dx, dgy, dw = fill(x.shape, dtype), fill(x.shape, dtype), fill(w.shape), up(x), up(gy), up(w)
    plan.forward(dx, dw, out)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw)
    gpu_device.sync()
    r, m = (o.conv(values(x[0]), values(w), grad=values(gy[0]), magnitude=q) for q in (False, True))
    o.within(values(out[0]), r["out"], m["out"], _rounds(width), dtype, "out")
    o.within(values(gx[0]), r["x"], m["x"], _rounds(width), dtype, "grad_x")
    o.within(values(gw), r["weight"], m["weight"], _rounds(width, length), "float32", "grad_weight")


# ------------------------------------------------------------- NaN and infinity


def _untouched(got, good, touched):
    """Bits outside `touched` are the same, and what is in it is NaN."""
    for k, t in touched.items():
        a, b = got[k].get(), good[k].get()
        assert same(a[~t], b[~t]), k
        assert torch.isnan(a[t]).all(), k


def _marks(**shapes):
    return {k: torch.zeros(s, dtype=torch.bool) for k, s in shapes.items()}


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("states,dtype", [(16, "float32"), (13, "float32"), (16, "bfloat16"), (24, "float16")])
def test_scan_gradients_of_nan(gpu_device, states, dtype, packed):
    """A NaN in u reaches its own channel's outputs, states and gradients, and
    B's and C's at the tokens where the sum over channels has a term with it; a
    NaN in the output's gradient the way back.  The rest keeps its bits."""
    import ferrum_gpu
    batch, length, channels, c, t, back = 2, 90, 40, 5, 50, 9
    i = _inputs(np.random.default_rng(3), (batch, length), channels, states, 1, dtype, batch)
    flat = (lambda v: v.flatten(0, 1)) if packed else (lambda v: v)
    off = {"offsets": up(torch.arange(0, 2 * length + 1, length, dtype=torch.int32))} if packed else {}
    plan = ferrum_gpu.ssm.ScanPlan(batch, length, channels, states, gpu_device, dtype=dtype,
                                   tokens=batch * length if packed else None)
    rows = ("u", "delta", "z", "B", "C", "gy")

    def run(j):
        d = {k: up(flat(v).contiguous() if k in rows else v) for k, v in j.items()}
        check = room(plan.checkpoint_bytes)
        got = {k: like(d[k]) for k in GRADS}
        got.update(out=like(d["u"]), final=like(d["initial"]), initial=like(d["initial"]))
        main, opt = [d[k] for k in MAIN], {k: d[k] for k in ("D", "z", "delta_bias")}
        plan.forward(*main, got["out"], **opt, initial=d["initial"], final=got["final"], checkpoints=check, **off)
        plan.backward(*main, d["gy"], check, **opt, **{"grad_" + k: got[k] for k in GRADS},
                      grad_initial=got["initial"], grad_final=d["gfinal"], **off)
        gpu_device.sync()
        return got

    good = run(i)
    shape, bc = (batch, length, channels), (batch, length, 1, states)
    marks = lambda: _marks(out=shape, final=(batch, channels, states), initial=(batch, channels, states),  # noqa: E731
                           u=shape, delta=shape, z=shape, B=bc, C=bc, A=(channels, states), D=(channels,),
                           delta_bias=(channels,))
    for key in ("u", "gy"):
        j = {k: v.clone() for k, v in i.items()}
        m = marks()
        if key == "u":
            j["u"][0, t, c] = float("nan")
            m["out"][0, t:, c] = m["z"][0, t:, c] = m["final"][0, c] = True
            m["delta"][0, t:, c] = True  # its own input at t, the states before later tokens
            m["B"][0, t] = True
            m["C"][0, t:] = True
        else:
            j["gy"][0, back, c] = float("nan")
            m["u"][0, :back + 1, c] = m["delta"][0, :back + 1, c] = m["initial"][0, c] = m["z"][0, back, c] = True
            m["B"][0, :back + 1] = True
            m["C"][0, back] = True
        m["A"][c] = m["D"][c] = m["delta_bias"][c] = True
        _untouched(run(j), good, {k: flat(v) if k in rows + ("out",) else v for k, v in m.items()})


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,channels", [("float32", 40), ("bfloat16", 40), ("float16", 37)])
def test_conv_of_nan(gpu_device, dtype, channels, packed):
    """A NaN in x reaches the outputs whose window holds it and the gradients
    of what these windows hold; one in the output's gradient its window's."""
    import ferrum_gpu
    rng = np.random.default_rng(4)
    batch, length, width, c, t = 2, 40, 4, 6, 17
    x, gy = (_rounded(rng, (batch, length, channels), dtype) for _ in range(2))
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    flat = (lambda v: v.flatten(0, 1)) if packed else (lambda v: v)
    off = {"offsets": up(torch.arange(0, 2 * length + 1, length, dtype=torch.int32))} if packed else {}
    plan = ferrum_gpu.ssm.ConvPlan(batch, length, channels, width, gpu_device, dtype=dtype,
                                   tokens=batch * length if packed else None)

    def run(x, gy):
        dx, dgy, dw = up(flat(x).contiguous()), up(flat(gy).contiguous()), up(w)
        got = dict(out=like(dx), x=like(dx), weight=like(dw), bias=fill((channels,)),
                   final=fill((batch, width - 1, channels), dtype))
        plan.forward(dx, dw, got["out"], final=got["final"], **off)
        plan.backward(dx, dw, dgy, grad_x=got["x"], grad_weight=got["weight"], grad_bias=got["bias"], **off)
        gpu_device.sync()
        return got

    good = run(x, gy)
    marks = lambda: _marks(out=x.shape, x=x.shape, weight=w.shape, bias=(channels,),  # noqa: E731
                           final=(batch, width - 1, channels))
    bad, m = x.clone(), marks()
    bad[0, t, c] = float("nan")
    m["out"][0, t:t + width, c] = m["x"][0, t - width + 1:t + width, c] = m["weight"][c] = m["bias"][c] = True
    _untouched(run(bad, gy), good, {k: flat(v) if k in ("out", "x") else v for k, v in m.items()})
    bad, m = gy.clone(), marks()
    bad[0, t, c] = float("nan")
    m["x"][0, t - width + 1:t + 1, c] = m["weight"][c] = m["bias"][c] = True
    _untouched(run(x, bad), good, {k: flat(v) if k in ("out", "x") else v for k, v in m.items()})
    # in a sequence's last rows: its final state, and nothing of the next sequence
    bad, m = x.clone(), marks()
    bad[0, length - 1, c] = float("nan")
    m["out"][0, length - 1, c] = m["final"][0, width - 2, c] = m["x"][0, length - width:, c] = True
    m["weight"][c] = m["bias"][c] = True
    _untouched(run(bad, gy), good, {k: flat(v) if k in ("out", "x") else v for k, v in m.items()})


@pytest.mark.parametrize("states,dtype", [(16, "float32"), (13, "bfloat16"), (64, "float16")])
def test_steps_of_nan(gpu_device, states, dtype):
    """A NaN in one row's input or state stays with that row and channel."""
    import ferrum_gpu
    ssm = ferrum_gpu.ssm
    rng, batch, channels, width, r, c = np.random.default_rng(5), 6, 40, 4, 2, 7
    i = _inputs(rng, (batch,), channels, states, 1, dtype, batch)
    window = _rounded(rng, (batch, width - 1, channels), dtype)
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()

    def run(i, window):
        d, win = {k: up(v) for k, v in i.items()}, up(window)
        got = dict(scan=like(d["u"]), state=like(d["initial"]), conv=like(d["u"]), window=like(win))
        ssm.scan_step(gpu_device, *(d[k] for k in MAIN), d["initial"], got["scan"], D=d["D"], z=d["z"],
                      delta_bias=d["delta_bias"], state_out=got["state"])
        ssm.conv_step(gpu_device, d["u"], up(w), win, got["conv"], state_out=got["window"])
        gpu_device.sync()
        return got

    good = run(i, window)
    marks = lambda: _marks(scan=(batch, channels), state=(batch, channels, states), conv=(batch, channels),  # noqa: E731
                           window=window.shape)
    j, m = {k: v.clone() for k, v in i.items()}, marks()
    j["u"][r, c] = float("nan")
    m["scan"][r, c] = m["state"][r, c] = m["conv"][r, c] = m["window"][r, width - 2, c] = True
    _untouched(run(j, window), good, m)
    j, m, bad = {k: v.clone() for k, v in i.items()}, marks(), window.clone()
    j["initial"][r, c, 1] = bad[r, 1, c] = float("nan")
    m["scan"][r, c] = m["state"][r, c, 1] = m["conv"][r, c] = m["window"][r, 0, c] = True
    _untouched(run(j, bad), good, m)


@pytest.mark.parametrize("batch,tokens,forward,backward", [
    (4, None, 4, 4), (5, None, 1, 4), (8, None, 1, 2), (9, None, 1, 1), (10, None, 1, 1), (15, None, 1, 1),
    (20, 4096, 8, 8), (20, 8192, 1, 4), (20, 12288, 1, 3), (20, 14336, 1, 1)])
def test_scan_parts_by_waves(gpu_device, batch, tokens, forward, backward):
    """Sequences of 128 waves each: the axis is cut where that was measured to gain."""
    import ferrum_gpu
    d = ferrum_gpu.ssm.ScanPlan(batch, 1024, 2048, 16, gpu_device, tokens=tokens).describe()
    assert (d["forward_parts"], d["backward_parts"]) == (forward, backward), d
