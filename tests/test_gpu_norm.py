"""The residual norm and dropout on the GPU against their definitions in 64 bits.

Tolerances.  u = 2^-24.  A thread sums its elements of a row one after another, a
team's threads in a tree: at most 200 + width / 64 roundings, the other steps of a
value a dozen more.  So normed values and gradients are held to (240 + width / 64) u
of the absolute values that they are sums of, the weight's gradient, a sum over
rows as well, to (240 + width / 64 + rows) u, and where rows are rounded to their
type, to half a step of it (e4m3: 2^-4, and 2^-10 below its normal numbers)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import ferrum_gpu
from ferrum_gpu import norm, pointwise
from ferrum_gpu.norm import NormPlan
from gpu_tensor import Gpu, fill, like, same, up, use, values

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
M = 2 ** 64 - 1


@pytest.fixture(autouse=True)
def on_device(gpu_device):
    yield from use(gpu_device)


def number(seed, j):
    """splitmix64's output j of a seed, in Python's integers."""
    z = (seed + (j + 1) * 0x9E3779B97F4A7C15) & M
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M
    return z ^ (z >> 31)


def kept(n, p, seed, offset):
    with np.errstate(over="ignore"):
        z = np.uint64(seed & M) + (np.arange((n + 1) // 2, dtype=np.uint64) + np.uint64((offset + 1) & M)) * \
            np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    bits = np.stack([z & np.uint64(0xFFFFFFFF), z >> np.uint64(32)], -1).reshape(-1)[:n].astype(np.float64)
    return torch.from_numpy(bits >= round(p * 2.0 ** 32))


def rows(shape, dtype, seed, scale=1.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    wide = (scale * torch.randn(shape[0], shape[1] + pad, generator=g)).to(TYPES[dtype])
    return wide[:, :shape[1]]


def half_step(dtype):
    return 0.0 if dtype == "float32" else torch.finfo(TYPES[dtype]).eps / 2


def near(got, want, by, what, dtype="float32", factor=240.0):
    got, want, by = values(got), want.numpy(), by.numpy()
    bound = factor * U * by
    least = 0 if dtype == "float32" else torch.finfo(TYPES[dtype]).tiny * torch.finfo(TYPES[dtype]).eps
    bound = bound + half_step(dtype) * (np.abs(want) + bound) + least + 1e-37
    off = np.abs(got - want)
    assert (off <= bound).all(), f"{what}: worst {np.max(off / bound):.2f} times the bound, {(~(off <= bound)).sum()} values"


def definition(x, residual, weight, eps, p=0.0, seed=0, offset=0):
    """v, out and what their errors go by."""
    v = x.double()
    if p:
        v = torch.where(kept(v.numel(), p, seed, offset).reshape(v.shape), v / (1 - p) if p < 1 else 0 * v, 0)
    size = v.abs()
    if residual is not None:
        v, size = v + residual.double(), size + residual.double().abs()
    s = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    w = torch.ones(x.shape[1], dtype=torch.float64) if weight is None else weight.double()
    return v, size, v * s * w, size * s * w.abs(), s


CASES = [(1, 1, "float32"), (3, 5, "bfloat16"), (2, 8, "float16"), (5, 63, "float32"), (1, 64, "bfloat16"),
         (7, 130, "bfloat16"), (4, 512, "float16"), (3, 520, "bfloat16"), (2, 1000, "float32"), (1, 1024, "bfloat16"),
         (5, 1025, "float16"), (3, 1500, "float16"), (2, 2048, "bfloat16"), (9, 2049, "float32"), (2, 4096, "bfloat16"),
         (3, 4099, "bfloat16"), (2, 8192, "float16"), (1, 8200, "float32"), (2, 16384, "bfloat16"), (2, 16392, "bfloat16"),
         (2, 40001, "float16"), (4100, 70, "bfloat16"), (2500, 1030, "bfloat16")]


@pytest.mark.parametrize("n,width,dtype", CASES)
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_forward_and_backward(gpu_device, n, width, dtype, p):
    x, residual = rows((n, width), dtype, 1), rows((n, width), dtype, 2, 3.0)
    weight = 1 + 0.3 * torch.randn(width)
    drop = {"dropout": p, "seed": 77, "offset": 1000}
    plan = NormPlan(n, width, gpu_device, dtype=dtype, eps=1e-5)
    out, total = fill((n, width), dtype), fill((n, width), dtype)
    plan.forward(up(x), out, weight=up(weight), residual=up(residual), sum_out=total, **drop)
    v, v_by, y, y_by, _ = definition(x, residual, weight, 1e-5, p, 77, 1000)
    f = 240 + width / 64
    near(total, v, v_by, "sum", dtype, 4)
    near(out, y, y_by, "out", dtype, f)
    # backward, from the sum as it was stored
    grad, grad_sum = rows((n, width), dtype, 3), rows((n, width), dtype, 4)
    gx, gr, gw = fill((n, width), dtype), fill((n, width), dtype), fill((width,))
    plan.backward(total, up(grad), weight=up(weight), grad_sum=up(grad_sum), grad_x=gx, grad_residual=gr,
                  grad_weight=gw, **drop)
    u = total.get().double()
    s = 1 / torch.sqrt((u * u).mean(-1, keepdim=True) + 1e-5)
    g = grad.double() * weight.double()
    dv = s * (g - u * s * s * (g * u).mean(-1, keepdim=True)) + grad_sum.double()
    by = s * (g.abs() + u.abs() * s * s * (g * u).abs().mean(-1, keepdim=True)) + grad_sum.double().abs()
    near(gr, dv, by, "grad_residual", dtype, f)
    mask = kept(n * width, p, 77, 1000).reshape(n, width) if p else torch.ones(n, width, dtype=torch.bool)
    near(gx, torch.where(mask, dv / (1 - p), 0), torch.where(mask, by / (1 - p), 0), "grad_x", dtype, f)
    terms = grad.double() * u * s
    near(gw, terms.sum(0), terms.abs().sum(0), "grad_weight", factor=f + n)


@pytest.mark.parametrize("n,width,dtype", [(1, 1, "bfloat16"), (3, 100, "float32"), (5, 130, "bfloat16"), (2, 513, "float16"),
                                           (3, 1500, "float16"), (4, 2048, "bfloat16"), (2, 4100, "float32"),
                                           (3, 4096, "bfloat16"), (2, 16400, "bfloat16"), (2, 9999, "float32")])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
def test_eight_bits(gpu_device, n, width, dtype, group):
    x, residual, weight = rows((n, width), dtype, 1), rows((n, width), dtype, 2), 1 + 0.3 * torch.randn(width)
    x[0, :min(width, 32)] = 0
    residual[0, :min(width, 32)] = 0
    plan = NormPlan(n, width, gpu_device, dtype=dtype, group=group)
    groups = -(-width // group) if group else 1
    out, scales, total = fill((n, width), "uint8"), fill((n, groups)), fill((n, width), dtype)
    plan.forward(up(x), out, weight=up(weight), residual=up(residual), sum_out=total, scales=scales)
    v, v_by, y, y_by, _ = definition(x, residual, weight, 1e-6)
    near(total, v, v_by, "sum", dtype, 4)
    f = (240 + width / 64) * U
    got, sc = out.get().view(torch.float8_e4m3fn).double(), values(scales)
    size = group or width
    for k in range(groups):
        part, by = y[:, k * size:(k + 1) * size], y_by[:, k * size:(k + 1) * size].max(-1).values.numpy()
        want = part.abs().max(-1).values.numpy() / 448
        assert (np.abs(sc[:, k] - want) <= f * by / 448 + 1e-37).all()
        q = got[:, k * size:(k + 1) * size].numpy()
        none = want == 0
        assert (sc[none, k] == 0).all() and (q[none] == 0).all()
        exact = part.numpy()[~none] / want[~none, None]
        slack = 3 * f * (by[~none] / want[~none])[:, None] / 1.0
        bound = 2.0 ** -4 * (np.abs(exact) + slack) + 2.0 ** -10 + slack
        assert (np.abs(q[~none] - exact) <= bound).all()
        assert (np.abs(q[~none]).max(-1) == 448).all()


@pytest.mark.parametrize("without", ["weight", "residual", "sum_out", "all"])
@pytest.mark.parametrize("width", [100, 2048, 17000])
def test_options(gpu_device, without, width):
    n, dtype = 3, "bfloat16"
    x, residual, weight = rows((n, width), dtype, 1, pad=3), rows((n, width), dtype, 2, pad=8), torch.randn(width)
    given = {"weight": weight, "residual": residual, "sum_out": fill((n, width), dtype)}
    for k in given:
        if without in (k, "all"):
            given[k] = None
    plan, out = NormPlan(n, width, gpu_device, dtype=dtype), fill((n, width + 4), dtype)
    plan.forward(up(x), out[:, :width], **{k: up(t) if isinstance(t, torch.Tensor) else t for k, t in given.items()})
    v, v_by, y, y_by, _ = definition(x, given["residual"], given["weight"], 1e-6)
    near(out[:, :width], y, y_by, "out", dtype, 240 + width / 64)
    assert (values(out)[:, width:] == 7).all()
    if given["sum_out"] is not None:
        near(given["sum_out"], v, v_by, "sum", dtype, 4)


@pytest.mark.parametrize("width", [130, 4096, 17001])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_in_place(gpu_device, width, p):
    """out over x and sum over the residual, gradients over those they come from, give what apart gives."""
    n, dtype = 5, "bfloat16"
    x, residual, weight = rows((n, width), dtype, 1), rows((n, width), dtype, 2), up(torch.randn(width))
    plan, drop = NormPlan(n, width, gpu_device, dtype=dtype), {"dropout": p, "seed": 5}
    out, total = fill((n, width), dtype), fill((n, width), dtype)
    plan.forward(up(x), out, weight=weight, residual=up(residual), sum_out=total, **drop)
    a, b = up(x), up(residual)
    plan.forward(a, a, weight=weight, residual=b, sum_out=b, **drop)
    assert same(a, out) and same(b, total)
    grad, grad_sum = rows((n, width), dtype, 3), rows((n, width), dtype, 4)
    gx, gr = fill((n, width), dtype), fill((n, width), dtype)
    plan.backward(total, up(grad), weight=weight, grad_sum=up(grad_sum), grad_x=gx, grad_residual=gr, **drop)
    a, b = up(grad), up(grad_sum)
    plan.backward(total, a, weight=weight, grad_sum=b, grad_x=a, grad_residual=b, **drop)
    assert same(a, gx) and same(b, gr)


def test_fewer_rows_and_none(gpu_device):
    """A call takes as many rows as x has, up to the plan's; rows behind them stay."""
    plan, weight = NormPlan(1000, 256, gpu_device), up(torch.randn(256))
    x = rows((700, 256), "bfloat16", 1)
    outs, d = [fill((700, 256), "bfloat16") for _ in range(2)], up(x)
    plan.forward(d, outs[0], weight=weight)
    plan.forward(d[:300], outs[1][:300], weight=weight)
    a, b = values(outs[0]), values(outs[1])
    assert np.array_equal(a[:300], b[:300]) and (b[300:] == 7).all()
    gw = [fill((256,)) for _ in range(3)]
    plan.backward(d, outs[0], weight=weight, grad_weight=gw[0])
    plan.backward(d[:300], outs[0][:300], weight=weight, grad_weight=gw[1])
    small = NormPlan(300, 256, gpu_device)
    small.backward(d[:300], outs[0][:300], weight=weight, grad_weight=gw[2])
    assert np.abs(values(gw[1]) - values(gw[2])).max() <= 600 * U * 300 * 16
    plan.forward(d[:0], outs[1][:0], weight=weight)
    plan.backward(d[:0], outs[0][:0], weight=weight, grad_weight=gw[1])
    assert (values(gw[1]) == 0).all()
    with pytest.raises(ferrum_gpu._native.FerrumGpuError, match="rows must be in"):
        small.forward(d[:301], outs[0][:301])


def test_same_bits_again(gpu_device):
    n, width = 3000, 1024
    x, grad, weight = up(rows((n, width), "bfloat16", 1)), up(rows((n, width), "bfloat16", 2)), up(torch.randn(width))
    plan, seen = NormPlan(n, width, gpu_device), None
    for _ in range(3):
        gw, gx = fill((width,)), fill((n, width), "bfloat16")
        plan.backward(x, grad, weight=weight, grad_x=gx, grad_weight=gw)
        now = (gw.get(), gx.get())
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, now))
        seen = now


def test_gradient_is_the_difference(gpu_device):
    """(f(x + e d) - f(x - e d)) / 2e with e = 2^-6 along the gradient: 1e-2 of its length covers the third
    derivative's e^2 / 6 and roundings of 500 u of sums over e."""
    n, width, e = 4, 200, 2.0 ** -6
    v = {"x": rows((n, width), "float32", 1), "residual": rows((n, width), "float32", 2), "weight": 1 + 0.2 * torch.randn(width)}
    grad, grad_sum = torch.randn(n, width), torch.randn(n, width)
    plan, drop = NormPlan(n, width, gpu_device, dtype="float32"), {"dropout": 0.25, "seed": 9}
    out, total = fill((n, width)), fill((n, width))

    def loss(w):
        plan.forward(up(w["x"]), out, weight=up(w["weight"]), residual=up(w["residual"]), sum_out=total, **drop)
        return ((out.get().double() * grad).sum() + (total.get().double() * grad_sum).sum()).item()

    loss(v)
    g = {k: like(t) for k, t in v.items()}
    plan.backward(total, up(grad), weight=up(v["weight"]), grad_sum=up(grad_sum), grad_x=g["x"],
                  grad_residual=g["residual"], grad_weight=g["weight"], **drop)
    for k in v:
        along = g[k].get() / g[k].get().norm()
        slope = (loss({**v, k: v[k] + e * along}) - loss({**v, k: v[k] - e * along})) / (2 * e)
        assert abs(slope / g[k].get().double().norm().item() - 1) < 1e-2, k


@pytest.mark.parametrize("group", [None, 0, 128])
def test_rows_that_are_not_finite_stay_alone(gpu_device, group):
    n, width = 6, 600
    x, weight = rows((n, width), "float32", 1), torch.randn(width)
    bad = x.clone()
    bad[1, 5], bad[3, 590], bad[4] = float("nan"), float("inf"), float("nan")
    outs = []
    for t in (x, bad):
        plan = NormPlan(n, width, gpu_device, dtype="float32", group=group or 0)
        out = fill((n, width), "float32" if group is None else "uint8")
        scales = None if group is None else fill((n, -(-width // group) if group else 1))
        plan.forward(up(t), out, weight=up(weight), scales=scales)
        got = values(out)
        if scales is not None:
            q = out.get().view(torch.float8_e4m3fn).double()
            got = (q * scales.get().double().repeat_interleave(group or width, 1)[:, :width]).numpy()
        outs.append(got)
    fine = [0, 2, 5]
    assert np.array_equal(outs[0][fine], outs[1][fine])
    assert np.isnan(outs[1][1]).all() and np.isnan(outs[1][4]).all() and np.isnan(outs[1][3, 590])


def test_empty_scales_and_large_values(gpu_device):
    """Rows of zeros have scales of 0; rows from 1e-25 to 1e15 fill their 8 bits."""
    width = 300
    x = torch.zeros(5, width)
    for k, s in ((1, 1e-25), (2, 1.0), (3, 1e15)):
        x[k] = s * torch.randn(width)
    plan = NormPlan(5, width, gpu_device, dtype="float32")
    out, scales = fill((5, width), "uint8"), fill((5, 1))
    plan.forward(up(x), out, scales=scales)
    q, s = out.get().view(torch.float8_e4m3fn).double(), scales.get().double()
    _, _, y, _, _ = definition(x, None, None, 1e-6)
    assert (q[[0, 4]] == 0).all() and (s[[0, 4]] == 0).all()
    assert (q[1:4].abs().max(-1).values == 448).all()
    assert ((q * s - y).abs()[1:4].max(-1).values <= 0.07 * y.abs()[1:4].max(-1).values).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 1000, 4097, 300001])
@pytest.mark.parametrize("p", [0.1, 0.75])
def test_dropout(gpu_device, dtype, n, p):
    x = torch.randn(n).to(TYPES[dtype])
    out = fill((n + 3,), dtype)
    pointwise.dropout(gpu_device, up(x), out[:n], n, p, 123, offset=55)
    want = torch.where(kept(n, p, 123, 55), x.double() / (1 - p), 0)
    near(out[:n], want, want.abs(), "out", dtype, 4)
    assert (values(out)[n:] == 7).all()
    inplace = up(x)
    pointwise.dropout(gpu_device, inplace, inplace, n, p, 123, offset=55)
    assert same(inplace, out[:n])


def test_dropout_bits_are_the_generators():
    assert [bool(v) for v in kept(64, 0.5, 3, 10)] == [
        (number(3, 10 + e // 2) >> (32 * (e % 2)) & 0xFFFFFFFF) >= 2 ** 31 for e in range(64)]


def test_dropout_of_part_of_a_tensor_continues(gpu_device):
    """A call behind another, its offset behind the numbers that that one used, is the rest of one call; and
    the count on the GPU is added to the offset."""
    n, cut = 4000, 1500
    x = torch.randn(n)
    whole, parts = fill((n,)), fill((n,))
    pointwise.dropout(gpu_device, up(x), whole, n, 0.4, 9, offset=2 ** 63)
    d = up(x)
    pointwise.dropout(gpu_device, d[:cut], parts[:cut], cut, 0.4, 9, offset=2 ** 63)
    pointwise.dropout(gpu_device, d[cut:], parts[cut:], n - cut, 0.4, 9, offset=2 ** 63 - 50,
                      counter=up(torch.tensor([cut // 2 + 50])))
    assert same(whole, parts)


@pytest.mark.parametrize("p", [0.0, 1e-12, 1.0])
def test_dropout_of_nothing_and_all(gpu_device, p):
    x = torch.randn(1001)
    x[5] = float("nan")
    out = fill((1001,))
    pointwise.dropout(gpu_device, up(x), out, 1001, p, 1)
    assert (values(out) == 0).all() if p == 1 else torch.equal(out.get().nan_to_num(1), x.nan_to_num(1))


def test_dropout_unaligned(gpu_device):
    """Any alignment of the elements."""
    x = torch.randn(1003).bfloat16()
    whole, d = fill((1003,), "bfloat16"), up(torch.cat([torch.zeros(1).bfloat16(), x]))
    pointwise.dropout(gpu_device, d[1:], whole, 1003, 0.2, 4)
    want = torch.where(kept(1003, 0.2, 4, 0), x.double() / 0.8, 0)
    near(whole, want, want.abs(), "out", "bfloat16", 4)


def test_captured_calls_replay(gpu_device):
    """A training step's norm and dropout in a graph, a count on the GPU moving the masks on."""
    n, width = 70, 520
    x, residual, grad = (Gpu(rows((n, width), "bfloat16", k)) for k in range(3))
    weight, counter = up(torch.randn(width)), up(torch.tensor([0]))
    plan = NormPlan(n, width, gpu_device)
    outs = [like(x.cpu) for _ in range(5)] + [fill((width,))]

    def calls(stream=0):
        drop = {"dropout": 0.2, "seed": 3, "counter": counter, "stream": stream}
        plan.forward(x, outs[0], weight=weight, residual=residual, sum_out=outs[1], **drop)
        plan.backward(outs[1], grad, weight=weight, grad_x=outs[2], grad_residual=outs[3], grad_weight=outs[5], **drop)
        pointwise.dropout(gpu_device, x, outs[4], n * width, 0.2, 4, counter=counter, stream=stream)

    with pytest.raises(ferrum_gpu._native.FerrumGpuError, match="first backward call"):
        with ferrum_gpu.hip.Capture(gpu_device) as cap:
            calls(cap.stream)
    calls()
    gpu_device.sync()
    with ferrum_gpu.hip.Capture(gpu_device, keep=[plan, outs]) as cap:
        calls(cap.stream)
    masks = []
    for k in range(4):
        x.normal_()
        counter.copy_(torch.tensor([1000 * k]))
        calls()
        gpu_device.sync()
        want = [t.get() for t in outs]
        for t in outs:
            t.fill_(7)
        cap.graph.launch()
        gpu_device.sync()
        assert all(torch.equal(a, t.get()) for a, t in zip(want, outs)), k
        masks.append(want[4] == 0)
    assert not torch.equal(masks[0], masks[1])


def test_rows_far_apart(gpu_device):
    """Rows whose offsets pass 32 bits: 2^25 elements between rows, 80 of them in one buffer of 5.4 GB."""
    from ferrum_gpu import _native as N
    n, width, row = 80, 200, 1 << 25
    x = rows((n, width), "bfloat16", 1).contiguous()
    buf = ferrum_gpu.hip.DeviceBuffer(gpu_device, 2 * ((n - 1) * row + 512))
    for r in range(n):
        N.check(N.lib.fg_copy_h2d(gpu_device.handle, buf.ptr + 2 * r * row, x[r].data_ptr(), 2 * width))

    class Rows:
        shape, dtype = x.shape, x.dtype
        def __init__(self, at): self.at = at
        def data_ptr(self): return buf.ptr + 2 * self.at
        def get_device(self): return gpu_device.ordinal
        def stride(self): return row, 1
        def is_contiguous(self): return False

    plan, outs = NormPlan(n, width, gpu_device), [fill((n, width), "bfloat16") for _ in range(3)]
    plan.forward(up(x), outs[0])
    plan.forward(Rows(0), outs[1])
    plan.forward(up(x), Rows(256))
    gpu_device.sync()
    for r in range(n):
        N.check(N.lib.fg_copy_d2h(gpu_device.handle, outs[2].cpu[r].data_ptr(), buf.ptr + 2 * (r * row + 256), 2 * width))
    assert same(outs[0], outs[1]) and torch.equal(outs[2].cpu, outs[0].get())
    buf.free()


def test_device_buffers_and_addresses(gpu_device):
    n, width = 5, 100
    x, residual = up(rows((n, width), "float32", 1)), up(rows((n, width), "float32", 2))
    outs = [fill((n, width)) for _ in range(2)]
    plan = NormPlan(n, width, gpu_device, dtype="float32")
    plan.forward(x, outs[0], residual=residual)
    plan.forward(x.buf, outs[1].data_ptr(), residual=residual.buf)
    assert same(*outs)
    plan.forward(x.buf, outs[1].buf, residual=residual.buf, rows=3)
    small = ferrum_gpu.hip.DeviceBuffer(gpu_device, 64)
    with pytest.raises(ValueError, match="buffer of 64 bytes"):
        plan.forward(x, small)


def test_refusals(gpu_device):
    n, width = 4, 256
    error = ferrum_gpu._native.FerrumGpuError
    plan = NormPlan(n, width, gpu_device)
    x, out, q = fill((n, width), "bfloat16"), fill((n, width), "bfloat16"), fill((n, width), "uint8")
    scales = fill((n, 1))
    for bad, why in ((dict(out=fill((n, width))), "float32"), (dict(residual=fill((n, 255), "bfloat16")), "shape"),
                     (dict(weight=fill((255,))), "shape"), (dict(scales=scales), "float8_e4m3fn"),
                     (dict(out=q, scales=fill((n, 2))), "shape"), (dict(counter=fill((1,), "int32")), "int32")):
        with pytest.raises(ValueError, match=why):
            plan.forward(**{**dict(x=x, out=out), **bad})
    for bad, why in ((dict(out=0), "null buffer"), (dict(dropout=1.5), "dropout"), (dict(dropout=float("nan")), "dropout"),
                     (dict(sum_out=x), "overlap"), (dict(out=x.data_ptr() + 2 * width), "overlap"),
                     (dict(sum_out=out), "overlap"), (dict(residual=x, out=x), "overlap")):
        with pytest.raises(error, match=why):
            plan.forward(**{**dict(x=x, out=out), **bad})
    with pytest.raises(error, match="overlap"):
        plan.backward(x, out, grad_x=x)
    for bad in (dict(width=0), dict(rows=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(group=48), dict(group=256)):
        with pytest.raises(error):
            NormPlan(**{**dict(rows=n, width=width, device=gpu_device), **bad})
    for bad, why in ((dict(p=-0.1), "dropout"), (dict(n=-1), "n must be"), (dict(out=x.data_ptr() + 2), "overlap")):
        with pytest.raises(error, match=why):
            pointwise.dropout(**{**dict(device=gpu_device, x=x, out=out, n=n * width, p=0.1, seed=0), **bad})
    for bad, why in ((dict(out=fill((n, width))), "float32"), (dict(n=n * width + 1), "contiguous bytes")):
        with pytest.raises(ValueError, match=why):
            pointwise.dropout(**{**dict(device=gpu_device, x=x, out=out, n=n * width, p=0.1, seed=0), **bad})
    plan.destroy()
    with pytest.raises(ValueError, match="destroyed"):
        plan.forward(x, out)
    assert norm.NormPlan is NormPlan
