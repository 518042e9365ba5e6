"""Run by test_gpu_ssm_streams.py in a process of its own, in which torch is
imported before the package: the sequence filters between torch operations on
torch's default stream, on a stream of its own and in a graph that torch captures,
without a wait of the host, against the same with one after every operation.

Every input is made behind work that takes milliseconds, over memory that held
other values: a call that did not wait for it would take those."""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrum-gpu_amd"))
import ferrum_gpu  # noqa: E402

ssm = ferrum_gpu.ssm
device = ferrum_gpu.hip.Device(0)
batch, length, channels, states, width = 2, 300, 96, 16, 4
conv = ssm.ConvPlan(batch, length, channels, width, device, dtype="float32")
scan = ssm.ScanPlan(batch, length, channels, states, device, dtype="float32")
source = {k: torch.randn(batch, length, n, device="cuda") for k, n in
          dict(x=channels, delta=channels, z=channels, B=states, C=states, grad=channels).items()}
held = {k: torch.empty_like(v) for k, v in source.items()}
w, A = torch.randn(channels, width, device="cuda"), -torch.rand(channels, states, device="cuda")
check = torch.empty(scan.checkpoint_bytes, dtype=torch.uint8, device="cuda")
u, y, gu, gx = (torch.empty(batch, length, channels, device="cuda") for _ in range(4))
gB, gA, gw = torch.empty_like(held["B"]), torch.empty_like(A), torch.empty_like(w)
window, state = torch.empty(batch, width - 1, channels, device="cuda"), torch.empty(batch, channels, states, device="cuda")
one, two = torch.empty(batch, channels, device="cuda"), torch.empty(batch, channels, device="cuda")
slow = torch.randn(2048, 2048, device="cuda")


def delay():
    s = slow
    for _ in range(20):
        s = s @ slow * 1e-2
    return s


def step(wait=lambda: None):
    """Torch operations and the filters in turn; returns copies of what they made."""
    here = torch.cuda.current_stream()
    extra = delay()
    for k in held:
        held[k].copy_(source[k])
        held[k].add_(extra[0, 0] * 0)
    wait()
    conv.forward(held["x"], w, u, final=window, stream=here)
    wait()
    v = u * 2
    wait()
    main = v, held["delta"], A, held["B"], held["C"]
    scan.forward(*main, y, z=held["z"], final=state, checkpoints=check, stream=here)
    scan.backward(*main, held["grad"], check, z=held["z"], grad_u=gu, grad_B=gB, grad_A=gA, stream=here)
    wait()
    g = gu * 2
    wait()
    conv.backward(held["x"], w, g, grad_x=gx, grad_weight=gw, stream=here)
    ssm.conv_step(device, y[:, 0], w, window, one, stream=here)
    wait()
    t = one + y[:, 1]
    wait()
    ssm.scan_step(device, t, held["delta"][:, 0], A, held["B"][:, 0], held["C"][:, 0], state, two, stream=here)
    wait()
    got = [x.clone() for x in (u, y, gu, gB, gA, gx, gw, window, state, one, two)]
    wait()
    return got


def spoil():
    for x in (*held.values(), u, y, gu, gx, gB, gA, gw, window, state, one, two):
        x.fill_(7)
    torch.cuda.synchronize()


def new_inputs():
    for x in source.values():
        x.normal_()
    torch.cuda.synchronize()


def compare(name, got, want):
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)), name
    print(f"{name}: same", flush=True)


def waiting():
    torch.cuda.synchronize()


for turn in range(3):
    new_inputs()
    spoil()
    want = step(waiting)
    spoil()
    compare(f"default stream {turn}", step(), want)
    spoil()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    compare(f"side stream {turn}", got, want)

spoil()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
for turn in range(4):
    new_inputs()
    spoil()
    want = step(waiting)
    spoil()
    graph.replay()
    compare(f"captured {turn}", captured, want)

try:
    other = type("Stream", (), {"cuda_stream": 0, "device_index": 1})()
    conv.forward(held["x"], w, u, stream=other)
except ValueError as e:
    assert "GPU 1" in str(e)
else:
    raise AssertionError("a stream of another GPU was taken")
print("done", flush=True)
