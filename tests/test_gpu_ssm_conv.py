"""The causal convolution on the GPU against its 64-bit oracle: whole sequences,
gradients, single tokens; layouts, packed sequences, states, refusals."""

from __future__ import annotations

import numpy as np
import pytest

import ssm_oracle as o

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import gpu_tensor  # noqa: E402
from gpu_tensor import Far, fill, like, same, up, values  # noqa: E402


@pytest.fixture(autouse=True)
def _on_gpu(gpu_device):
    yield from gpu_tensor.use(gpu_device)


def _type(dtype):
    return getattr(torch, dtype)


def _rounded(rng, shape, dtype, scale=1.0):
    return (torch.from_numpy(rng.standard_normal(shape)) * scale).to(_type(dtype))


def _rounds(width, summed=1):
    # products and sums of the taps, the bias, the activation and its slope (at most 30 between them)
    return 2 * width + summed + 32


def _check(dev, rng, batch, length, channels, width, dtype, silu=True, bias=True, state=True, layout="plain"):
    """Forward and backward of one dense call in a layout."""
    import ferrum_gpu
    x, gy = (_rounded(rng, (batch, length, channels), dtype) for _ in range(2))
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    b = torch.from_numpy(rng.standard_normal(channels)).float() if bias else None
    ini, gf = ((_rounded(rng, (batch, width - 1, channels), dtype) if state else None) for _ in range(2))

    def laid(v, room=False):
        v = torch.full_like(v, 7) if room else v
        if layout == "window":    # a column window of a wider array
            big = torch.full(v.shape[:2] + (2 * channels + 3,), 7.0, dtype=v.dtype)
            big[..., channels + 1:2 * channels + 1] = v
            return up(big[..., channels + 1:2 * channels + 1])
        if layout == "tokens":    # tokens before sequences
            return up(v.transpose(0, 1).contiguous().transpose(0, 1))
        return up(v)

    dx, dgy, out, gx = laid(x), laid(gy), laid(x, True), laid(x, True)
    fin, gini = (fill((batch, width - 1, channels), dtype) if state else None for _ in range(2))
    gw, gb = fill((channels, width), "float32"), fill((channels,), "float32")
    dw, db, dini, dgf = up(w), up(b), up(ini), up(gf)
    plan = ferrum_gpu.ssm.ConvPlan(batch, length, channels, width, dev, dtype=dtype,
                                   activation="silu" if silu else None)
    plan.forward(dx, dw, out, bias=db, initial=dini, final=fin)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw, grad_bias=gb, bias=db, initial=dini, grad_initial=gini,
                  grad_final=dgf)
    dev.sync()
    tw, tb = np.zeros((channels, width)), np.zeros(channels)
    mw, mb = tw.copy(), tb.copy()
    for s in range(batch):
        args = dict(x=values(x[s]), w=values(w), bias=None if b is None else values(b), initial=None if ini is None else
                    values(ini[s]), silu=silu, grad=values(gy[s]), grad_final=None if gf is None else values(gf[s]))
        r, m = o.conv(**args), o.conv(**args, magnitude=True)
        o.within(values(out[s]), r["out"], m["out"], _rounds(width), dtype, "out")
        o.within(values(gx[s]), r["x"], m["x"], _rounds(width), dtype, "grad_x")
        if state:
            assert np.array_equal(values(fin[s]), r["final"])
            o.within(values(gini[s]), r["initial"], m["initial"], _rounds(width), dtype, "grad_initial")
        tw, tb, mw, mb = tw + r["weight"], tb + r["bias"], mw + m["weight"], mb + m["bias"]
    o.within(values(gw), tw, mw, _rounds(width, batch * length), "float32", "grad_weight")
    o.within(values(gb), tb, mb, _rounds(width, batch * length), "float32", "grad_bias")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("batch,length,channels,width", [
    (1, 1, 8, 4), (2, 2, 64, 4), (3, 3, 7, 2), (1, 5, 513, 3), (2, 33, 96, 4), (2, 16, 1, 8), (1, 70, 520, 5),
    (2, 131, 24, 6), (1, 64, 260, 7), (4, 17, 128, 8), (1, 1030, 8, 4)])
def test_sizes(gpu_device, batch, length, channels, width, dtype):
    print(f"[case] conv {batch}x{length}x{channels} width={width} {dtype}", flush=True)
    _check(gpu_device, np.random.default_rng(length * 10 + width), batch, length, channels, width, dtype)


@pytest.mark.parametrize("layout", ["plain", "window", "tokens"])
@pytest.mark.parametrize("silu,bias,state", [(True, False, False), (False, True, True), (False, False, False)])
def test_layouts_and_options(gpu_device, layout, silu, bias, state):
    print(f"[case] conv layout={layout} silu={silu} bias={bias} state={state}", flush=True)
    _check(gpu_device, np.random.default_rng(5), 3, 37, 72, 4, "bfloat16", silu, bias, state, layout)


@pytest.mark.parametrize("channels", [40, 37])
def test_packed(gpu_device, channels):
    """Empty, one-token and longer sequences, rows before, between and after
    them that belong to none (NaN there reaches nothing; outputs stay as they
    were), and offsets that are out of order or beyond the rows."""
    import ferrum_gpu
    rng = np.random.default_rng(11)
    width, tokens, longest = 4, 90, 33
    offsets = [2, 2, 3, 36, 36, 38, 80]  # the last is longer than the plan's length: cut
    used = [(2, 2), (2, 3), (3, 36), (36, 36), (36, 38), (38, 38 + longest)]
    x, gy = (_rounded(rng, (tokens, channels), "float32") for _ in range(2))
    for v in (x, gy):
        v[:2] = v[38 + longest:] = float("nan")
    w, b = torch.from_numpy(rng.standard_normal((channels, width))).float(), torch.zeros(channels)
    ini = _rounded(rng, (len(used), width - 1, channels), "float32")
    plan = ferrum_gpu.ssm.ConvPlan(len(used), longest, channels, width, gpu_device, dtype="float32", tokens=tokens)
    off = up(torch.tensor(offsets, dtype=torch.int32))
    out, gx, fin = fill(x.shape, "float32"), fill(x.shape, "float32"), fill(ini.shape, "float32")
    gw = fill(w.shape, "float32")
    dx, dgy, dw, db, dini = up(x), up(gy), up(w), up(b), up(ini)
    plan.forward(dx, dw, out, bias=db, initial=dini, final=fin, offsets=off)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw, bias=db, initial=dini, offsets=off)
    gpu_device.sync()
    tw, mw = 0, 0
    touched = np.zeros(tokens, bool)
    for s, (i, j) in enumerate(used):
        touched[i:j] = True
        args = dict(x=values(x[i:j]), w=values(w), bias=values(b), initial=values(ini[s]), grad=values(gy[i:j]))
        r, m = o.conv(**args), o.conv(**args, magnitude=True)
        o.within(values(out[i:j]), r["out"], m["out"], _rounds(width), "float32", "out")
        o.within(values(gx[i:j]), r["x"], m["x"], _rounds(width), "float32", "grad_x")
        assert np.array_equal(values(fin[s]), r["final"])
        tw, mw = tw + r["weight"], mw + m["weight"]
    o.within(values(gw), tw, mw, _rounds(width, tokens), "float32", "grad_weight")
    assert all((v.get()[torch.from_numpy(~touched)] == 7).all() for v in (out, gx))
    # taken as the nearest valid ones: rows -5 .. 4 are 0 .. 4, 60 .. 500 are 60 .. 90, and 500 .. 60 are none
    off.copy_(torch.tensor([-5, 4, 60, 500, 60, 60, 60], dtype=torch.int32))
    out.fill_(7)
    plan.forward(dx, dw, out, bias=db, initial=dini, offsets=off)
    gpu_device.sync()
    want = o.conv(values(x[4:60][:longest]), values(w), values(b), values(ini[1]))["out"]
    assert np.allclose(values(out[4:4 + longest]), want, rtol=1e-4, atol=1e-4)
    assert (out[4 + longest:60] == 7).all()


@pytest.mark.parametrize("longest", [700, 21])
def test_packed_parameter_gradients(gpu_device, longest):
    """Many short sequences and a plan for much longer ones, or for shorter
    ones (which cuts them): nothing of an earlier call's other sequences, rows
    before, between or after is in the sums."""
    import ferrum_gpu
    rng = np.random.default_rng(23)
    width, tokens, channels, n = 4, 700, 24, 30
    x, gy = (_rounded(rng, (tokens, channels), "float32") for _ in range(2))
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    plan = ferrum_gpu.ssm.ConvPlan(n, longest, channels, width, gpu_device, dtype="float32", tokens=tokens)
    gw, gb, dx, dgy, dw = fill(w.shape), fill((channels,)), up(x), up(gy), up(w)
    for start, most in ((0, 46), (17, 30), (300, 3)):
        lengths = np.minimum(rng.integers(0, most, n), tokens)
        offsets = np.minimum(start + np.concatenate([[0], np.cumsum(lengths)]), tokens).astype(np.int32)
        plan.backward(dx, dw, dgy, grad_weight=gw, grad_bias=gb, offsets=up(torch.from_numpy(offsets)))
        gpu_device.sync()
        want, size = [0, 0], [0, 0]
        for i, j in zip(offsets[:-1], np.minimum(offsets[1:], offsets[:-1] + longest)):
            r, m = (o.conv(values(x[i:j]), values(w), grad=values(gy[i:j]), magnitude=q) for q in (False, True))
            want = [want[0] + r["weight"], want[1] + r["bias"]]
            size = [size[0] + m["weight"], size[1] + m["bias"]]
        o.within(values(gw), want[0], size[0], _rounds(width, tokens), "float32", "grad_weight")
        o.within(values(gb), want[1], size[1], _rounds(width, tokens), "float32", "grad_bias")


def test_no_tokens(gpu_device):
    """No sequences, or sequences without tokens: states pass through, parameter gradients are zeros."""
    import ferrum_gpu
    w = up(torch.ones(8, 3))
    for batch, length in ((0, 5), (2, 0)):
        x = fill((batch, length, 8))
        ini = up(torch.randn(batch, 2, 8))
        fin, gini, gw = fill((batch, 2, 8), "float32"), fill((batch, 2, 8), "float32"), fill((8, 3), "float32")
        plan = ferrum_gpu.ssm.ConvPlan(batch, length, 8, 3, gpu_device, dtype="float32")
        plan.forward(x, w, like(x), initial=ini, final=fin)
        plan.backward(x, w, like(x), grad_weight=gw, initial=ini, grad_initial=gini, grad_final=ini)
        gpu_device.sync()
        assert same(fin, ini) and same(gini, ini) and (gw == 0).all()


def test_final_may_be_initial(gpu_device):
    import ferrum_gpu
    x = up(torch.randn(2, 1, 64))
    state = up(torch.randn(2, 4, 64))
    want = torch.cat([state.get(), x.get()], 1)[:, 1:]
    w, out = up(torch.randn(64, 5)), like(x)
    plan = ferrum_gpu.ssm.ConvPlan(2, 1, 64, 5, gpu_device, dtype="float32")
    plan.forward(x, w, out, initial=state, final=state)
    gpu_device.sync()
    assert same(state, want)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("width", [2, 5, 6, 7, 8])
def test_final_may_be_initial_over_runs(gpu_device, width, packed):
    """Several runs to a sequence: none but the first may read the state."""
    import ferrum_gpu
    batch, length, channels = 16, 61, 200
    tokens = batch * length
    x = up(torch.randn(*((tokens,) if packed else (batch, length)), channels))
    state = up(torch.randn(batch, width - 1, channels))
    kept, fin, w = state.clone(), fill((batch, width - 1, channels), "float32"), up(torch.randn(channels, width))
    a, b = like(x), like(x)
    off = {"offsets": up(torch.arange(0, tokens + 1, length, dtype=torch.int32))} if packed else {}
    plan = ferrum_gpu.ssm.ConvPlan(batch, length, channels, width, gpu_device, dtype="float32",
                                   tokens=tokens if packed else None)
    plan.forward(x, w, a, initial=kept, final=fin, **off)
    plan.forward(x, w, b, initial=state, final=state, **off)
    gpu_device.sync()
    assert same(a, b) and same(fin, state)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("batch,channels,width", [(1, 8, 4), (5, 1000, 4), (3, 65, 3), (2, 2048, 8), (7, 16, 2)])
def test_step(gpu_device, batch, channels, width, dtype):
    """Slots in any order, one row without a slot and one beyond the windows;
    the windows of no row stay as they are."""
    import ferrum_gpu
    rng = np.random.default_rng(batch * 100 + width)
    rows = batch + 3
    x, st = _rounded(rng, (batch, channels), dtype), _rounded(rng, (rows, width - 1, channels), dtype)
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    b = torch.from_numpy(rng.standard_normal(channels)).float()
    slots = rng.permutation(rows)[:batch].astype(np.int32)
    if batch > 2:
        slots[0], slots[1] = -1, rows
    for in_place in (True, False):
        dst, out = up(st), fill((batch, channels), dtype)
        new = None if in_place else dst.clone()
        wide = fill((batch, 2 * channels), dtype)
        wide[:, channels:] = x
        args = up(w), up(b), up(torch.from_numpy(slots))
        ferrum_gpu.ssm.conv_step(gpu_device, wide[:, channels:], args[0], dst, out, bias=args[1], slots=args[2],
                                 state_out=new)
        gpu_device.sync()
        want_state = values(st)
        for i, s in enumerate(slots):
            if s < 0 or s >= rows:
                assert (out[i] == 0).all()
                continue
            a = dict(x=values(x[i])[None], w=values(w), bias=values(b), initial=values(st[s]))
            r, m = o.conv(**a), o.conv(**a, magnitude=True)
            o.within(values(out[i]), r["out"][0], m["out"][0], _rounds(width), dtype, "out")
            want_state[s] = r["final"]
        assert np.array_equal(values(dst if in_place else new), want_state)
        if not in_place:
            assert same(dst, st)


def test_long_runs_and_many_rows(gpu_device):
    """Tokens enough for a thread's longest run forward, and rows enough for a
    wave to walk through several."""
    import ferrum_gpu
    rng = np.random.default_rng(31)
    length, channels, width = 270001, 8, 4
    x, gy = (_rounded(rng, (1, length, channels), "float32") for _ in range(2))
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    out, gx, gw = fill(x.shape, "float32"), fill(x.shape, "float32"), fill(w.shape, "float32")
    dx, dgy, dw = up(x), up(gy), up(w)
    plan = ferrum_gpu.ssm.ConvPlan(1, length, channels, width, gpu_device, dtype="float32")
    rows = fill((length, channels))
    state = _rounded(rng, (length, width - 1, channels), "float32")
    before, state = state, up(state)
    new = like(state)
    plan.forward(dx, dw, out)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw)
    ferrum_gpu.ssm.conv_step(gpu_device, dx[0], dw, state, rows, state_out=new)
    gpu_device.sync()
    r, m = (o.conv(values(x[0]), values(w), grad=values(gy[0]), magnitude=q) for q in (False, True))
    o.within(values(out[0]), r["out"], m["out"], _rounds(width), "float32", "out")
    o.within(values(gx[0]), r["x"], m["x"], _rounds(width), "float32", "grad_x")
    # the sums run in parts: at most 64 tokens, then eight running sums of the parts in each of four waves
    o.within(values(gw), r["weight"], m["weight"], _rounds(width, length), "float32", "grad_weight")
    win = np.concatenate([values(before), values(x[0])[:, None]], 1)
    p, mp = ((q(win) * q(values(w)).T).sum(1) for q in (lambda v: v, np.abs))
    o.within(values(rows), p * o.sigmoid(p), mp, _rounds(width), "float32", "step")
    assert np.array_equal(values(new), win[:, 1:]) and same(state, before)


def test_windows_of_one_array(gpu_device):
    """One token of each row: input and output that are columns of one array."""
    import ferrum_gpu
    big = up(torch.randn(3, 1, 64))
    w, st = up(torch.randn(32, 4)), up(torch.randn(3, 3, 32))
    want, new = fill((3, 1, 32)), like(st)
    plan = ferrum_gpu.ssm.ConvPlan(3, 1, 32, 4, gpu_device, dtype="float32")
    plan.forward(up(big.get()[..., :32].contiguous()), w, want, initial=st)
    plan.forward(big[..., :32], w, big[..., 32:], initial=st)
    gpu_device.sync()
    assert same(big[..., 32:], want)
    ferrum_gpu.ssm.conv_step(gpu_device, big[:, 0, :32], w, st, big[:, 0, 32:], state_out=new)
    gpu_device.sync()
    assert same(big[..., 32:], want)


def test_prompt_then_tokens(gpu_device):
    """A prompt and single tokens after it are the whole sequence."""
    import ferrum_gpu
    batch, length, channels, width, more = 2, 9, 48, 4, 5
    x = up(torch.randn(batch, length + more, channels))
    w = up(torch.randn(channels, width))
    whole, out = like(x), like(x)
    state = fill((batch, width - 1, channels))
    ssm = ferrum_gpu.ssm
    ssm.ConvPlan(batch, length + more, channels, width, gpu_device, dtype="float32").forward(x, w, whole)
    plan = ssm.ConvPlan(batch, length, channels, width, gpu_device, dtype="float32")
    plan.forward(x[:, :length], w, out[:, :length], final=state)
    for t in range(length, length + more):
        ssm.conv_step(gpu_device, x[:, t], w, state, out[:, t])
    gpu_device.sync()
    assert same(out, whole)


def test_refusals(gpu_device):
    import ferrum_gpu
    from ferrum_gpu import _native as N
    ssm, E = ferrum_gpu.ssm, N.FerrumGpuError
    make = lambda **k: ssm.ConvPlan(**{**dict(batch=2, length=8, channels=16, width=4, device=gpu_device,  # noqa: E731
                                              dtype="float32"), **k})
    for bad in (dict(width=1), dict(width=9), dict(channels=0), dict(batch=-1), dict(length=-1)):
        with pytest.raises(E, match="must be in"):
            make(**bad)
    with pytest.raises(ValueError, match="dtype"):
        make(dtype="float64")
    plan = make()
    x, out = up(torch.zeros(2, 8, 16)), up(torch.zeros(2, 8, 16))
    w, b = up(torch.zeros(16, 4)), up(torch.zeros(16))
    st = up(torch.zeros(2, 3, 16))
    big = up(torch.zeros(2, 8, 32))
    with pytest.raises(ValueError, match="shape"):
        plan.forward(x[:, :7], w, out)
    with pytest.raises(ValueError, match="runs on GPU"):
        plan.forward(x.get(), w, out)
    with pytest.raises(ValueError, match="only packed"):
        plan.forward(x, w, out, offsets=up(torch.zeros(3, dtype=torch.int32)))
    with pytest.raises(ValueError, match="packed sequences need them"):
        make(tokens=16).forward(x.view(16, 16), w, out.view(16, 16))
    with pytest.raises(E, match="overlap"):
        plan.forward(x, w, x)
    with pytest.raises(E, match="overlap"):
        plan.forward(x, w, out[:1].expand(2, 8, 16))
    with pytest.raises(E, match="overlap"):
        plan.forward(big[..., :16], w, big[..., 8:24])
    plan.forward(big[..., :16], w, big[..., 16:])  # windows side by side are apart
    with pytest.raises(E, match="overlap"):
        plan.backward(x, w, out, grad_x=big[..., :16], grad_weight=w)
    with pytest.raises(ValueError, match="float32"):
        plan.forward(x, up(w.get().half()), out)
    with pytest.raises(E, match="null buffer"):
        plan.forward(0, w, out)
    with pytest.raises(E, match="not aligned"):
        plan.forward(x.data_ptr() + 2, w, out)
    with pytest.raises(E, match="exceeds"):
        make(batch=1, length=2, channels=(1 << 25) + 8, width=2).forward(x.data_ptr(), w.data_ptr(), out.data_ptr())
    with pytest.raises(E, match="too large"):
        make(batch=(1 << 31) - 1, channels=1 << 25, width=8)
    with pytest.raises(E, match="too large"):
        ssm.conv_step(gpu_device, x.data_ptr(), w.data_ptr(), st.data_ptr(), out.data_ptr(), batch=2,
                      channels=(1 << 31) - 1, width=8, state_rows=(1 << 31) - 1, dtype="float32")
    with pytest.raises(ValueError, match="bytes"):
        plan.forward(ferrum_gpu.hip.DeviceBuffer(gpu_device, 64), w, out)
    with pytest.raises(E, match="state_rows"):
        ssm.conv_step(gpu_device, x[:, 0], w, st[:1], out[:, 0])
    with pytest.raises(E, match="overlap"):
        ssm.conv_step(gpu_device, x[:, 0], w, st, out[:, 0], state_out=x.view(-1)[:96].view(2, 3, 16))
    with pytest.raises(ValueError, match="needed"):
        ssm.conv_step(gpu_device, x.data_ptr(), w, st, out[:, 0])
    plan.destroy()
    with pytest.raises(ValueError, match="destroyed"):
        plan.forward(x, w, out)
    gpu_device.sync()


def test_device_buffers_and_addresses(gpu_device):
    """The package's own buffers, without torch's types."""
    import ferrum_gpu
    from ferrum_gpu.hip import DeviceBuffer
    rng = np.random.default_rng(2)
    x, w = rng.standard_normal((3, 5, 8)).astype(np.float32), rng.standard_normal((8, 4)).astype(np.float32)
    dx, dw, dy, ds = (DeviceBuffer(gpu_device, n) for n in (x.nbytes, w.nbytes, x.nbytes, 3 * 3 * 8 * 4))
    dx.copy_from_host(x)
    dw.copy_from_host(w)
    plan = ferrum_gpu.ssm.ConvPlan(3, 5, 8, 4, gpu_device, dtype="float32", activation=None)
    plan.forward(dx, dw.ptr, dy, final=ds)
    got = dy.copy_to_host(np.empty_like(x))
    for s in range(3):
        r, m = (o.conv(x[s].astype(float), w.astype(float), silu=False, magnitude=q) for q in (False, True))
        o.within(got[s], r["out"], m["out"], _rounds(4), "float32", "out")
    step = np.empty((3, 8), np.float32)
    dt, do = DeviceBuffer(gpu_device, step.nbytes), DeviceBuffer(gpu_device, step.nbytes)
    ferrum_gpu.ssm.conv_step(gpu_device, dt, dw, ds, do, activation=None, batch=3, channels=8, width=4, state_rows=3,
                             dtype="float32")
    do.copy_to_host(step)
    want = (x[:, 2:].transpose(0, 2, 1).astype(float) * w[:, :3]).sum(-1)
    assert np.allclose(step, want, rtol=1e-5, atol=1e-5)


def test_captured_calls_replay(gpu_device):
    """Forward, backward and a step in a graph, replayed with other inputs."""
    import ferrum_gpu
    from ferrum_gpu.hip import Capture
    from ferrum_gpu._native import FerrumGpuError
    ssm = ferrum_gpu.ssm
    x, gy = up(torch.randn(2, 40, 64)), up(torch.randn(2, 40, 64))
    w, st = up(torch.randn(64, 4)), up(torch.randn(2, 3, 64))
    out, gx, gw = like(x), like(x), like(w)
    so, new = fill((2, 64)), like(st)
    plan = ssm.ConvPlan(2, 40, 64, 4, gpu_device, dtype="float32")

    def calls(stream=0):
        plan.forward(x, w, out, initial=st, stream=stream)
        plan.backward(x, w, gy, grad_x=gx, grad_weight=gw, initial=st, stream=stream)
        ssm.conv_step(gpu_device, x[:, 0], w, st, so, state_out=new, stream=stream)

    with pytest.raises(FerrumGpuError, match="cannot be captured"):
        with Capture(gpu_device) as cap:
            calls(cap.stream)
    calls()
    with Capture(gpu_device, keep=[plan]) as cap:
        calls(cap.stream)
    for k in range(4):
        x.normal_()
        gy.normal_()
        calls()
        gpu_device.sync()
        want = [v.clone() for v in (out, gx, gw, so, new)]
        for v in (out, gx, gw, so, new):
            v.fill_(7)
        cap.graph.launch()
        gpu_device.sync()
        assert all(same(a, b) for a, b in zip(want, (out, gx, gw, so, new))), k


def test_rows_far_apart(gpu_device):
    """Rows whose distance from the first passes 2^32 bytes."""
    import ferrum_gpu
    from ferrum_gpu.hip import DeviceBuffer
    row, length = 1 << 25, 70
    x = torch.randn(1, length, 64).half()
    far, near = Far(DeviceBuffer(gpu_device, 2 * length * row), x, row, 0), up(x)
    w = up(torch.randn(64, 4))
    a, b = like(near), like(near)
    plan = ferrum_gpu.ssm.ConvPlan(1, length, 64, 4, gpu_device, dtype="float16")
    plan.forward(far, w, a)
    plan.forward(near, w, b)
    plan.forward(near, w, far)
    gpu_device.sync()
    assert same(a, b) and same(far, b)


def test_sizes_that_pass_64_bits(gpu_device):
    """Rows of stride 0 can stand for any number of them: no size worked out from it wraps around."""
    import ferrum_gpu
    from ferrum_gpu import _native as N
    ssm, E, most = ferrum_gpu.ssm, N.FerrumGpuError, (1 << 31) - 1
    for make in (lambda **k: ssm.ConvPlan(width=2, **k), lambda **k: ssm.ScanPlan(states=4, **k)):
        with pytest.raises(E, match="rows: too large"):
            make(batch=most, length=most, channels=1024, device=gpu_device)
        with pytest.raises(E, match="rows: too large"):
            make(batch=1, length=most, channels=1 << 25, tokens=1 << 40, device=gpu_device)
    # a workspace that no memory holds: 2^24 sequences' parts of 3 * 2^21 sums
    tokens, channels = 1 << 24, 1 << 21
    plan = ssm.ConvPlan(tokens, most, channels, 2, gpu_device, tokens=tokens)
    row = up(torch.zeros(1, channels, dtype=torch.bfloat16)).expand(tokens, channels)
    off = up(torch.zeros(tokens + 1, dtype=torch.int32))
    with pytest.raises(E, match="workspace: too large"):
        plan.backward(row, up(torch.zeros(channels, 2)), row, offsets=off)
    gpu_device.sync()


@pytest.mark.parametrize("lead", [(4, 9), (9, 4), (1, 9), (4, 1)])
def test_windows_of_an_array_with_tokens_first(gpu_device, lead):
    """Input and output, and two gradients, as columns of one (tokens,
    sequences, channels) array; windows that share a column are refused."""
    import ferrum_gpu
    from ferrum_gpu._native import FerrumGpuError
    batch, length = lead
    big = up(torch.randn(length, batch, 80).transpose(0, 1))
    a, b, shared = big[..., :32], big[..., 40:72], big[..., 71:]
    x, w, gy = up(a.get().contiguous()), up(torch.randn(32, 4)), up(torch.randn(batch, length, 32))
    want, out, gx = like(x), like(x), like(x)
    plan = ferrum_gpu.ssm.ConvPlan(batch, length, 32, 4, gpu_device, dtype="float32")
    plan.forward(x, w, want)
    plan.forward(a, w, b)
    gpu_device.sync()
    assert same(b, want)
    plan.backward(x, w, gy, grad_x=want)
    plan.backward(a, w, gy, grad_x=b)
    gpu_device.sync()
    assert same(b, want)
    small = ferrum_gpu.ssm.ConvPlan(batch, length, 9, 4, gpu_device, dtype="float32")
    for bad in (big[..., 63:72], big[..., 70:79]):
        with pytest.raises(FerrumGpuError, match="overlap"):
            small.forward(shared, up(torch.randn(9, 4)), bad)
    small.forward(shared, up(torch.randn(9, 4)), big[..., 62:71])
    scan = ferrum_gpu.ssm.ScanPlan(batch, length, 8, 4, gpu_device, dtype="float32")
    check = gpu_tensor.room(scan.checkpoint_bytes)
    u, B, C, A = big[..., :8], big[..., 8:12], big[..., 12:16], up(-torch.ones(8, 4))
    scan.forward(u, u, A, B, C, big[..., 16:24], checkpoints=check)
    scan.backward(u, u, A, B, C, big[..., 16:24], check, grad_u=big[..., 24:32], grad_delta=big[..., 32:40],
                  grad_B=big[..., 40:44], grad_C=big[..., 44:48])
    with pytest.raises(FerrumGpuError, match="grad_u and grad_delta overlap"):
        scan.backward(u, u, A, B, C, big[..., 16:24], check, grad_u=big[..., 24:32], grad_delta=big[..., 31:39])
    gpu_device.sync()
