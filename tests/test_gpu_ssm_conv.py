"""The causal convolution on the GPU against its 64-bit oracle: whole sequences,
gradients, single tokens; layouts, packed sequences, states, refusals."""

from __future__ import annotations

import numpy as np
import pytest

import ssm_oracle as o

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _type(dtype):
    return getattr(torch, dtype)


def _rounded(rng, shape, dtype, scale=1.0):
    return (torch.from_numpy(rng.standard_normal(shape)) * scale).to(_type(dtype))


def _np(x):
    return x.detach().double().cpu().numpy()


def _rounds(width, summed=1):
    # products and sums of the taps, the bias, the activation and its slope (at most 30 between them)
    return 2 * width + summed + 32


def _fill(shape, dtype, value=7.0):
    return torch.full(shape, value, dtype=_type(dtype), device="cuda")


def _done(dev):
    dev.sync()
    torch.cuda.synchronize()


def _check(dev, rng, batch, length, channels, width, dtype, silu=True, bias=True, state=True, layout="plain"):
    """Forward and backward of one dense call in a layout."""
    import ferrum_gpu
    x, gy = (_rounded(rng, (batch, length, channels), dtype) for _ in range(2))
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    b = torch.from_numpy(rng.standard_normal(channels)).float() if bias else None
    ini, gf = ((_rounded(rng, (batch, width - 1, channels), dtype) if state else None) for _ in range(2))

    def laid(v, room=False):
        v = v.cuda() if not room else _fill(v.shape, dtype)
        if layout == "window":    # a column window of a wider array
            big = _fill(v.shape[:2] + (2 * channels + 3,), dtype)
            big[..., channels + 1:2 * channels + 1] = v
            return big[..., channels + 1:2 * channels + 1]
        if layout == "tokens":    # tokens before sequences
            return v.transpose(0, 1).contiguous().transpose(0, 1)
        return v

    dx, dgy, out, gx = laid(x), laid(gy), laid(x, True), laid(x, True)
    fin, gini = (_fill((batch, width - 1, channels), dtype) if state else None for _ in range(2))
    gw, gb = _fill((channels, width), "float32"), _fill((channels,), "float32")
    cuda = lambda v: None if v is None else v.cuda()  # noqa: E731
    dw, db, dini, dgf = cuda(w), cuda(b), cuda(ini), cuda(gf)
    plan = ferrum_gpu.ssm.ConvPlan(batch, length, channels, width, dev, dtype=dtype,
                                   activation="silu" if silu else None)
    torch.cuda.synchronize()
    plan.forward(dx, dw, out, bias=db, initial=dini, final=fin)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw, grad_bias=gb, bias=db, initial=dini, grad_initial=gini,
                  grad_final=dgf)
    _done(dev)
    tw, tb = np.zeros((channels, width)), np.zeros(channels)
    mw, mb = tw.copy(), tb.copy()
    for s in range(batch):
        args = dict(x=_np(x[s]), w=_np(w), bias=None if b is None else _np(b), initial=None if ini is None else
                    _np(ini[s]), silu=silu, grad=_np(gy[s]), grad_final=None if gf is None else _np(gf[s]))
        r, m = o.conv(**args), o.conv(**args, magnitude=True)
        o.within(_np(out[s]), r["out"], m["out"], _rounds(width), dtype, "out")
        o.within(_np(gx[s]), r["x"], m["x"], _rounds(width), dtype, "grad_x")
        if state:
            assert np.array_equal(_np(fin[s]), r["final"])
            o.within(_np(gini[s]), r["initial"], m["initial"], _rounds(width), dtype, "grad_initial")
        tw, tb, mw, mb = tw + r["weight"], tb + r["bias"], mw + m["weight"], mb + m["bias"]
    o.within(_np(gw), tw, mw, _rounds(width, batch * length), "float32", "grad_weight")
    o.within(_np(gb), tb, mb, _rounds(width, batch * length), "float32", "grad_bias")


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
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out, gx, fin = _fill(x.shape, "float32"), _fill(x.shape, "float32"), _fill(ini.shape, "float32")
    gw = _fill(w.shape, "float32")
    dx, dgy, dw, db, dini = x.cuda(), gy.cuda(), w.cuda(), b.cuda(), ini.cuda()
    torch.cuda.synchronize()
    plan.forward(dx, dw, out, bias=db, initial=dini, final=fin, offsets=off)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw, bias=db, initial=dini, offsets=off)
    _done(gpu_device)
    tw, mw = 0, 0
    touched = np.zeros(tokens, bool)
    for s, (i, j) in enumerate(used):
        touched[i:j] = True
        args = dict(x=_np(x[i:j]), w=_np(w), bias=_np(b), initial=_np(ini[s]), grad=_np(gy[i:j]))
        r, m = o.conv(**args), o.conv(**args, magnitude=True)
        o.within(_np(out[i:j]), r["out"], m["out"], _rounds(width), "float32", "out")
        o.within(_np(gx[i:j]), r["x"], m["x"], _rounds(width), "float32", "grad_x")
        assert np.array_equal(_np(fin[s]), r["final"])
        tw, mw = tw + r["weight"], mw + m["weight"]
    o.within(_np(gw), tw, mw, _rounds(width, tokens), "float32", "grad_weight")
    assert (out[~torch.from_numpy(touched).cuda()] == 7).all() and (gx[~torch.from_numpy(touched).cuda()] == 7).all()
    # taken as the nearest valid ones: rows -5 .. 4 are 0 .. 4, 60 .. 500 are 60 .. 90, and 500 .. 60 are none
    off.copy_(torch.tensor([-5, 4, 60, 500, 60, 60, 60], dtype=torch.int32))
    out.fill_(7)
    torch.cuda.synchronize()
    plan.forward(dx, dw, out, bias=db, initial=dini, offsets=off)
    _done(gpu_device)
    want = o.conv(_np(x[4:60][:longest]), _np(w), _np(b), _np(ini[1]))["out"]
    assert np.allclose(_np(out[4:4 + longest]), want, rtol=1e-4, atol=1e-4)
    assert (out[4 + longest:60] == 7).all()


def test_no_tokens(gpu_device):
    """No sequences, or sequences without tokens: states pass through, parameter gradients are zeros."""
    import ferrum_gpu
    w = torch.ones(8, 3, device="cuda")
    for batch, length in ((0, 5), (2, 0)):
        x = torch.empty(batch, length, 8, device="cuda")
        ini = torch.randn(batch, 2, 8, device="cuda")
        fin, gini, gw = _fill((batch, 2, 8), "float32"), _fill((batch, 2, 8), "float32"), _fill((8, 3), "float32")
        plan = ferrum_gpu.ssm.ConvPlan(batch, length, 8, 3, gpu_device, dtype="float32")
        torch.cuda.synchronize()
        plan.forward(x, w, torch.empty_like(x), initial=ini, final=fin)
        plan.backward(x, w, torch.empty_like(x), grad_weight=gw, initial=ini, grad_initial=gini, grad_final=ini)
        _done(gpu_device)
        assert torch.equal(fin, ini) and torch.equal(gini, ini) and (gw == 0).all()


def test_final_may_be_initial(gpu_device):
    import ferrum_gpu
    x = torch.randn(2, 1, 64, device="cuda")
    state = torch.randn(2, 4, 64, device="cuda")
    want = torch.cat([state, x], 1)[:, 1:]
    w, out = torch.randn(64, 5, device="cuda"), torch.empty_like(x)
    plan = ferrum_gpu.ssm.ConvPlan(2, 1, 64, 5, gpu_device, dtype="float32")
    torch.cuda.synchronize()
    plan.forward(x, w, out, initial=state, final=state)
    _done(gpu_device)
    assert torch.equal(state, want)


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
        dst, out = st.cuda(), _fill((batch, channels), dtype)
        new = None if in_place else dst.clone()
        wide = _fill((batch, 2 * channels), dtype)
        wide[:, channels:] = x
        args = w.cuda(), b.cuda(), torch.from_numpy(slots).cuda()
        torch.cuda.synchronize()
        ferrum_gpu.ssm.conv_step(gpu_device, wide[:, channels:], args[0], dst, out, bias=args[1], slots=args[2],
                                 state_out=new)
        _done(gpu_device)
        want_state = _np(st)
        for i, s in enumerate(slots):
            if s < 0 or s >= rows:
                assert (out[i] == 0).all()
                continue
            a = dict(x=_np(x[i])[None], w=_np(w), bias=_np(b), initial=_np(st[s]))
            r, m = o.conv(**a), o.conv(**a, magnitude=True)
            o.within(_np(out[i]), r["out"][0], m["out"][0], _rounds(width), dtype, "out")
            want_state[s] = r["final"]
        assert np.array_equal(_np(dst if in_place else new), want_state)
        if not in_place:
            assert torch.equal(dst.cpu(), st)


def test_long_runs_and_many_rows(gpu_device):
    """Tokens enough for a thread's longest run forward, and rows enough for a
    wave to walk through several."""
    import ferrum_gpu
    rng = np.random.default_rng(31)
    length, channels, width = 270001, 8, 4
    x, gy = (_rounded(rng, (1, length, channels), "float32") for _ in range(2))
    w = torch.from_numpy(rng.standard_normal((channels, width))).float()
    out, gx, gw = _fill(x.shape, "float32"), _fill(x.shape, "float32"), _fill(w.shape, "float32")
    dx, dgy, dw = x.cuda(), gy.cuda(), w.cuda()
    plan = ferrum_gpu.ssm.ConvPlan(1, length, channels, width, gpu_device, dtype="float32")
    rows = torch.empty(length, channels, device="cuda")
    state = _rounded(rng, (length, width - 1, channels), "float32").cuda()
    before, new = state.clone(), torch.empty_like(state)
    torch.cuda.synchronize()
    plan.forward(dx, dw, out)
    plan.backward(dx, dw, dgy, grad_x=gx, grad_weight=gw)
    ferrum_gpu.ssm.conv_step(gpu_device, dx[0], dw, state, rows, state_out=new)
    _done(gpu_device)
    r, m = (o.conv(_np(x[0]), _np(w), grad=_np(gy[0]), magnitude=q) for q in (False, True))
    o.within(_np(out[0]), r["out"], m["out"], _rounds(width), "float32", "out")
    o.within(_np(gx[0]), r["x"], m["x"], _rounds(width), "float32", "grad_x")
    # the sums run in parts: at most 64 tokens, then eight running sums of the parts in each of four waves
    o.within(_np(gw), r["weight"], m["weight"], _rounds(width, length), "float32", "grad_weight")
    win = np.concatenate([_np(before), _np(x[0])[:, None]], 1)
    p, mp = ((q(win) * q(_np(w)).T).sum(1) for q in (lambda v: v, np.abs))
    o.within(_np(rows), p * o.sigmoid(p), mp, _rounds(width), "float32", "step")
    assert np.array_equal(_np(new), win[:, 1:]) and torch.equal(state, before)


def test_windows_of_one_array(gpu_device):
    """One token of each row: input and output that are columns of one array."""
    import ferrum_gpu
    big = torch.randn(3, 1, 64, device="cuda")
    w, st = torch.randn(32, 4, device="cuda"), torch.randn(3, 3, 32, device="cuda")
    want, new = torch.empty(3, 1, 32, device="cuda"), torch.empty_like(st)
    plan = ferrum_gpu.ssm.ConvPlan(3, 1, 32, 4, gpu_device, dtype="float32")
    torch.cuda.synchronize()
    plan.forward(big[..., :32].contiguous(), w, want, initial=st)
    plan.forward(big[..., :32], w, big[..., 32:], initial=st)
    _done(gpu_device)
    assert torch.equal(big[..., 32:], want)
    ferrum_gpu.ssm.conv_step(gpu_device, big[:, 0, :32], w, st, big[:, 0, 32:], state_out=new)
    _done(gpu_device)
    assert torch.equal(big[..., 32:], want)


def test_prompt_then_tokens(gpu_device):
    """A prompt and single tokens after it are the whole sequence."""
    import ferrum_gpu
    batch, length, channels, width, more = 2, 9, 48, 4, 5
    x = torch.randn(batch, length + more, channels, device="cuda")
    w = torch.randn(channels, width, device="cuda")
    whole, out = torch.empty_like(x), torch.empty_like(x)
    state = torch.empty(batch, width - 1, channels, device="cuda")
    ssm = ferrum_gpu.ssm
    torch.cuda.synchronize()
    ssm.ConvPlan(batch, length + more, channels, width, gpu_device, dtype="float32").forward(x, w, whole)
    plan = ssm.ConvPlan(batch, length, channels, width, gpu_device, dtype="float32")
    plan.forward(x[:, :length], w, out[:, :length], final=state)
    for t in range(length, length + more):
        ssm.conv_step(gpu_device, x[:, t], w, state, out[:, t])
    _done(gpu_device)
    assert torch.equal(out, whole)


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
    x, out = torch.zeros(2, 8, 16, device="cuda"), torch.zeros(2, 8, 16, device="cuda")
    w, b = torch.zeros(16, 4, device="cuda"), torch.zeros(16, device="cuda")
    st = torch.zeros(2, 3, 16, device="cuda")
    big = torch.zeros(2, 8, 32, device="cuda")
    with pytest.raises(ValueError, match="shape"):
        plan.forward(x[:, :7], w, out)
    with pytest.raises(ValueError, match="runs on GPU"):
        plan.forward(x.cpu(), w, out)
    with pytest.raises(ValueError, match="only packed"):
        plan.forward(x, w, out, offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
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
        plan.forward(x, w.half(), out)
    with pytest.raises(E, match="null buffer"):
        plan.forward(0, w, out)
    with pytest.raises(E, match="not aligned"):
        plan.forward(x.data_ptr() + 2, w, out)
    with pytest.raises(E, match="exceeds"):
        make(batch=1, length=2, channels=(1 << 25) + 8, width=2).forward(x.data_ptr(), w.data_ptr(), out.data_ptr())
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
    _done(gpu_device)


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
    x, gy = torch.randn(2, 40, 64, device="cuda"), torch.randn(2, 40, 64, device="cuda")
    w, st = torch.randn(64, 4, device="cuda"), torch.randn(2, 3, 64, device="cuda")
    out, gx, gw = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w)
    so, new = torch.empty(2, 64, device="cuda"), torch.empty_like(st)
    plan = ssm.ConvPlan(2, 40, 64, 4, gpu_device, dtype="float32")

    def calls(stream=0):
        plan.forward(x, w, out, initial=st, stream=stream)
        plan.backward(x, w, gy, grad_x=gx, grad_weight=gw, initial=st, stream=stream)
        ssm.conv_step(gpu_device, x[:, 0], w, st, so, state_out=new, stream=stream)

    torch.cuda.synchronize()
    with pytest.raises(FerrumGpuError, match="cannot be captured"):
        with Capture(gpu_device) as cap:
            calls(cap.stream)
    calls()
    with Capture(gpu_device, keep=[plan]) as cap:
        calls(cap.stream)
    for k in range(4):
        x.normal_()
        gy.normal_()
        torch.cuda.synchronize()
        calls()
        _done(gpu_device)
        want = [v.clone() for v in (out, gx, gw, so, new)]
        for v in (out, gx, gw, so, new):
            v.fill_(7)
        torch.cuda.synchronize()
        cap.graph.launch()
        _done(gpu_device)
        assert all(torch.equal(a, b) for a, b in zip(want, (out, gx, gw, so, new))), k


def test_rows_far_apart(gpu_device):
    """Rows whose distance from the first passes 2^32 bytes."""
    import ferrum_gpu
    row, length = 1 << 25, 70
    far = torch.empty(length * row, dtype=torch.float16, device="cuda").as_strided((1, length, 64), (0, row, 1))
    near = torch.randn(1, length, 64, device="cuda").half()
    far.copy_(near)
    w = torch.randn(64, 4, device="cuda")
    a, b = torch.empty_like(near), torch.empty_like(near)
    plan = ferrum_gpu.ssm.ConvPlan(1, length, 64, 4, gpu_device, dtype="float16")
    torch.cuda.synchronize()
    plan.forward(far, w, a)
    plan.forward(near, w, b)
    plan.forward(near, w, far)
    _done(gpu_device)
    assert torch.equal(a, b) and torch.equal(far.contiguous(), b)
