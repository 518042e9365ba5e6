"""The recurrence on the GPU where what it is given is at the edge of what it takes: offsets that fall, states in
one array, parameters that are not finite, arrays large enough for the kernels that pass the caches."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ferrum_gpu import ssm
from gpu_tensor import fill, room, same, up, use, values
from test_gpu_recurrence import TYPES, inputs, run

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_device(gpu_device):
    yield from use(gpu_device)


@pytest.mark.parametrize("dtype,channels", [("bfloat16", 64), ("float32", 37)])
@pytest.mark.parametrize("tokens,offsets", [
    (20, [0, 20, 5]), (20, [10, 20, 5]), (40, [9, 5, 40, 1, 1]), (700, [0, 600, 590, 700, 20]),
    (90, [-4, 2, 9, 5, 2 ** 31 - 1, 1, 1, 1]), (700, [700, 0, 700, 0])])
def test_falling_offsets_leave_what_lies_around(gpu_device, dtype, channels, tokens, offsets):
    """Outputs are undefined; what is in front of and behind every array of states and of checkpoints stays."""
    n = len(offsets) - 1
    v = inputs((tokens,), channels, dtype)
    d = {k: up(t) for k, t in v.items()}
    at = up(torch.tensor(offsets, dtype=torch.int32))
    plan = ssm.RecurrencePlan(n, tokens, channels, gpu_device, dtype=dtype, tokens=tokens)
    around = [fill((n + 4, channels)) for _ in range(4)]
    initial, final, grad_final, grad_initial = (a[2:n + 2] for a in around)
    check = room(plan.checkpoint_bytes + 4096)
    out, dx = fill((tokens + 4, channels), dtype), fill((tokens + 4, channels), dtype)
    main = (d["x"], d["gate_a"], d["gate_x"], d["decay"])
    grad = up(torch.randn(tokens, channels).to(TYPES[dtype]))
    plan.forward(*main, out[2:tokens + 2], initial=initial, final=final, offsets=at, checkpoints=check)
    plan.backward(*main, grad, check, grad_x=dx[2:tokens + 2], grad_final=grad_final, grad_initial=grad_initial, offsets=at)
    gpu_device.sync()
    assert (check.get()[plan.checkpoint_bytes:] == 0).all()
    for a in (*around, out, dx):
        got = values(a)
        assert np.all(got[:2] == 7) and np.all(got[-2:] == 7)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("length", [20, 100, 256, 600, 1300])
def test_states_in_one_array_carry_on(gpu_device, dtype, length):
    """Call after call takes its first states where it leaves its last ones, as calls with two arrays do."""
    lead, ch = (3, length), 132
    d = {k: up(t) for k, t in inputs(lead, ch, dtype).items()}
    main = (d["x"], d["gate_a"], d["gate_x"], d["decay"])
    plan = ssm.RecurrencePlan(*lead, ch, gpu_device, dtype=dtype)
    start = torch.randn(3, ch)
    one, turns = up(start), [up(start), fill((3, ch))]
    outs = [fill((*lead, ch), dtype) for _ in range(2)]
    for _ in range(8):
        plan.forward(*main, outs[0], initial=one, final=one)
        plan.forward(*main, outs[1], initial=turns[0], final=turns[1])
        turns.reverse()
        assert same(*outs) and same(one, turns[0])


@pytest.mark.parametrize("dtype,channels", [("float32", 64), ("bfloat16", 62)])
def test_one_token_is_a_sequence_of_one_whatever_the_parameters(gpu_device, dtype, channels):
    """Infinite decays, biases and gates: the step gives what a plan gives for one token, and a closed gate leaves
    the state in both."""
    rows, inf = 60, float("inf")
    v = inputs((rows,), channels, dtype)
    far = torch.tensor([inf, -inf, 0.5])
    for k, lead in (("decay", ()), ("bias_a", ()), ("bias_x", ()), ("gate_a", (rows,)), ("gate_x", (rows,))):
        v[k] = far[torch.randint(0, 3, (*lead, channels))].to(v[k].dtype)
    d = {k: up(t) for k, t in v.items()}
    state = torch.randn(rows, channels)
    outs, ends = [fill((rows, channels), dtype) for _ in range(2)], [fill((rows, channels)) for _ in range(2)]
    ssm.recurrence_step(gpu_device, **d, state=up(state), out=outs[0], state_out=ends[0])
    plan = ssm.RecurrencePlan(rows, 1, channels, gpu_device, dtype=dtype)
    seq = {k: d[k].view(rows, 1, channels) for k in ("x", "gate_a", "gate_x")}
    plan.forward(**{**d, **seq}, out=outs[1].view(rows, 1, channels), initial=up(state), final=ends[1])
    for a, b, step in ((*outs, 0 if dtype == "float32" else torch.finfo(TYPES[dtype]).eps), (*ends, 0)):
        a, b = values(a), values(b)
        # the same formula in float32: a dozen roundings of 2^-24, and a half step of the rows on either side
        assert np.array_equal(np.isnan(a), np.isnan(b))
        assert (np.abs(a - b) <= (12 * 2.0 ** -24 + step) * np.abs(b))[~np.isnan(b)].all()
    closed = (v["gate_a"] == -inf).numpy()
    assert np.array_equal(values(ends[0])[closed], state.double().numpy()[closed])


LARGE = 16 << 20  # bytes of rows from which on a plan takes the kernels that pass the caches


@pytest.mark.parametrize("batch,length,channels,dtype,layout", [
    (1, 1030, 8192, "bfloat16", "plain"), (2, 1100, 4098, "float16", "plain"), (3, 700, 2050, "float32", "windows"),
    (1, 2100, 4000, "bfloat16", "windows")])
def test_large_arrays(gpu_device, batch, length, channels, dtype, layout):
    assert batch * length * channels * TYPES[dtype].itemsize >= LARGE
    run(gpu_device, (batch, length), channels, dtype, layout=layout)


@pytest.mark.parametrize("channels,dtype,offsets", [
    (8194, "bfloat16", [0, 300, 300, 310, 1030]), (4100, "float16", [2, 700, 701, 702, 2100]),
    (4096, "float32", [0, 0, 33, 1024, 1030, 1100])])
def test_large_packed_arrays(gpu_device, channels, dtype, offsets):
    assert offsets[-1] * channels * TYPES[dtype].itemsize >= LARGE
    run(gpu_device, (offsets[-1] + 9,), channels, dtype, offsets=offsets)
