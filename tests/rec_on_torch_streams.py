"""Run by test_gpu_recurrent_layer.py in a process of its own, in which torch is
imported before the package: the recurrence, the norm and dropout between torch
operations on torch's default stream, on a stream of its own and in a graph that
torch captures, without a wait of the host, against the same with one after
every operation; and two plans at a time on two streams.

Every input is made behind work that takes milliseconds, over memory that held
other values: a call that did not wait for it would take those."""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrum-gpu_amd"))
import ferrum_gpu  # noqa: E402
from ferrum_gpu import pointwise, ssm  # noqa: E402
from ferrum_gpu.norm import NormPlan  # noqa: E402

device = ferrum_gpu.hip.Device(0)
batch, length, channels = 2, 700, 200
shape = (batch, length, channels)
plan = ssm.RecurrencePlan(*shape, device, dtype="float32")
norm = NormPlan(batch * length, channels, device, dtype="float32")
source = {k: torch.randn(shape, device="cuda") for k in ("x", "a", "i", "residual", "grad")}
held = {k: torch.empty_like(v) for k, v in source.items()}
p = torch.randn(channels, device="cuda")
check = torch.empty(plan.checkpoint_bytes, dtype=torch.uint8, device="cuda")
outs = {k: torch.empty(shape, device="cuda") for k in ("normed", "sum", "h", "dx", "da", "di", "dn", "dr", "dropped")}
sums = {k: torch.empty(channels, device="cuda") for k in ("decay", "weight")}
state, one = torch.empty(batch, channels, device="cuda"), torch.empty(batch, channels, device="cuda")
counter = torch.zeros(1, dtype=torch.int64, device="cuda")
slow = torch.randn(2048, 2048, device="cuda")


def delay():
    s = slow
    for _ in range(20):
        s = s @ slow * 1e-2
    return s


def rows(x):
    return x.view(-1, channels)


def step(wait=lambda: None):
    """Torch operations and the package's in turn; returns copies of what they made."""
    here = torch.cuda.current_stream()
    drop = {"dropout": 0.3, "seed": 5, "counter": counter, "stream": here}
    extra = delay()
    for k in held:
        held[k].copy_(source[k])
        held[k].add_(extra[0, 0] * 0)
    counter.add_(3)
    wait()
    norm.forward(rows(held["x"]), rows(outs["normed"]), weight=p, residual=rows(held["residual"]),
                 sum_out=rows(outs["sum"]), **drop)
    wait()
    v = outs["normed"] * 2
    wait()
    args = v, held["a"], held["i"], p
    plan.forward(*args, outs["h"], final=state, checkpoints=check, stream=here)
    plan.backward(*args, held["grad"], check, grad_x=outs["dx"], grad_gate_a=outs["da"], grad_gate_x=outs["di"],
                  grad_decay=sums["decay"], stream=here)
    wait()
    g = outs["dx"] * 2
    wait()
    norm.backward(rows(outs["sum"]), rows(g), weight=p, grad_x=rows(outs["dn"]), grad_residual=rows(outs["dr"]),
                  grad_weight=sums["weight"], **drop)
    pointwise.dropout(device, outs["h"], outs["dropped"], outs["h"].numel(), 0.5, 9, counter=counter, stream=here)
    ssm.recurrence_step(device, held["x"][:, 0], held["a"][:, 0], held["i"][:, 0], p, state, one, stream=here)
    wait()
    got = [x.clone() for x in (*outs.values(), *sums.values(), state, one)]
    wait()
    return got


def spoil():
    for x in (*held.values(), *outs.values(), *sums.values(), state, one):
        x.fill_(7)
    counter.zero_()
    torch.cuda.synchronize()


def new_inputs():
    for x in source.values():
        x.normal_()
    torch.cuda.synchronize()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def expected():
    spoil()
    want = step(lambda: torch.cuda.synchronize())
    spoil()
    return want


for name, where in (("default stream", torch.cuda.default_stream()), ("a stream", torch.cuda.Stream())):
    for k in range(3):
        new_inputs()
        want = expected()
        with torch.cuda.stream(where):
            got = step()
        torch.cuda.synchronize()
        assert same(got, want), (name, k)
    print(name, flush=True)

side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.stream(side):
    step()
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=side):
    got = step()
for k in range(4):
    new_inputs()
    want = expected()
    graph.replay()
    torch.cuda.synchronize()
    assert same(got, want), ("graph", k)
print("graph", flush=True)

# two plans of their own at a time: each has its own tickets and words
plans = [ssm.RecurrencePlan(*shape, device, dtype="float32") for _ in range(2)]
ways = [torch.cuda.Stream() for _ in range(2)]
xs = [[torch.randn(shape, device="cuda") for _ in range(3)] for _ in range(2)]
two, alone = [torch.empty(shape, device="cuda") for _ in range(2)], [torch.empty(shape, device="cuda") for _ in range(2)]
for k in range(2):
    plans[k].forward(*xs[k], p, alone[k], stream=torch.cuda.current_stream())
torch.cuda.synchronize()
for _ in range(20):
    for k in range(2):
        plans[k].forward(*xs[k], p, two[k], stream=ways[k])
torch.cuda.synchronize()
assert same(two, alone)
print("two at a time", flush=True)
print("done", flush=True)
