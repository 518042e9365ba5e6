"""The example layer of the recurrence, the residual norm and dropout: a prompt,
the same tokens one by one from a cache of slots, and its gradients; and the three
operators on torch's streams."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")

HERE = os.path.dirname(os.path.abspath(__file__))


def test_layer(gpu_device):
    """In a process of its own, with torch's tensors on the GPU: torch finds
    none where the package was loaded before it.  float32: about 60 tokens of
    some ten roundings each leave 1e-4 at most; e4m3 rounds by 2^-4 at most, 0.04 of
    the norm on average; the slope's step of 1e-2 leaves its square and rounding of
    1e-6 / 1e-2."""
    at = os.path.join(os.path.dirname(HERE), "ferrum-gpu_amd", "examples", "recurrent_layer.py")
    ran = subprocess.run([sys.executable, at], capture_output=True, text=True, timeout=100)
    assert ran.returncode == 0, ran.stderr
    got = dict(line.split(": ") for line in ran.stdout.splitlines())
    assert float(got["tokens against the whole"]) <= 1e-4
    assert float(got["8 bits against the rows' type"]) <= 2 ** -4
    assert float(got["slope against the gradient of y"]) <= 1e-2
    assert float(got["slope against the gradient of stream"]) <= 1e-2


def test_calls_follow_torchs_streams(gpu_device):
    at = os.path.join(HERE, "rec_on_torch_streams.py")
    ran = subprocess.run([sys.executable, at], capture_output=True, text=True, timeout=100)
    assert ran.returncode == 0, ran.stdout + ran.stderr
    assert ran.stdout.splitlines()[-1] == "done"


FIRST_CALLS = """
import sys
import numpy as np
sys.path.insert(0, sys.argv[1])
import ferrum_gpu
from ferrum_gpu.hip import Capture, Device, DeviceBuffer
dev, rng = Device(0), np.random.default_rng(0)
rows, channels = 3, 32

def up(x):
    b = DeviceBuffer(dev, x.nbytes)
    b.copy_from_host(x)
    return b

for dtype, of in (("float16", np.float16), ("float32", np.float32)):
    x = rng.standard_normal((rows, channels)).astype(of)
    p, h = (rng.standard_normal(s).astype(np.float32) for s in (channels, (rows, channels)))
    d, places = [up(v) for v in (x, p, h)], (x, h, x)
    outs = [up(np.full_like(v, 7)) for v in places]

    def calls(stream):
        ferrum_gpu.ssm.recurrence_step(dev, d[0], d[0], d[0], d[1], d[2], outs[0], state_out=outs[1], batch=rows,
                                       channels=channels, state_rows=rows, dtype=dtype, stream=stream)
        ferrum_gpu.pointwise.dropout(dev, d[0], outs[2], rows * channels, 0.5, 1, dtype=dtype, stream=stream)

    def results():
        return [o.copy_to_host(np.empty_like(v)) for o, v in zip(outs, places)]

    with Capture(dev) as cap:  # the first calls of this type in the process
        calls(cap.stream)
    got = []
    for _ in range(3):
        cap.graph.launch()
        got.append(results())
        for o, v in zip(outs, places):
            o.copy_from_host(np.full_like(v, 7))
    calls(0)
    want = results()
    assert all(np.array_equal(p, q) for g in got for p, q in zip(g, want)), dtype
    assert all(not (v == 7).all() for v in want)
    print(dtype, "same", flush=True)
"""


def test_a_types_first_call_may_be_captured(gpu_device):
    """In a process of its own, whose first call of a type loads its code object."""
    root = os.path.join(os.path.dirname(HERE), "ferrum-gpu_amd")
    ran = subprocess.run([sys.executable, "-c", FIRST_CALLS, root], capture_output=True, text=True, timeout=100)
    assert ran.returncode == 0, ran.stdout + ran.stderr
    assert ran.stdout.split() == ["float16", "same", "float32", "same"]
