"""The sequence filters on torch's streams, between torch's own operations."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")


def test_calls_follow_torchs_streams(gpu_device):
    """In a process of its own: torch finds no GPU where the package was loaded before it."""
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "ssm_on_torch_streams.py")
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
rows, channels, states, width = 3, 32, 16, 4

def up(x):
    b = DeviceBuffer(dev, x.nbytes)
    b.copy_from_host(x)
    return b

for dtype, of in (("float16", np.float16), ("float32", np.float32)):
    make = lambda *s: rng.standard_normal(s).astype(of)
    x, window = make(rows, channels), make(rows, width - 1, channels)
    w = rng.standard_normal((channels, width)).astype(np.float32)
    a, h = -np.ones((channels, states), np.float32), rng.standard_normal((rows, channels, states)).astype(np.float32)
    bc = make(rows, states)
    d = [up(v) for v in (x, w, window, a, bc, h)]
    outs = [up(np.full_like(v, 7)) for v in (x, window, x, h)]

    def calls(stream):
        ferrum_gpu.ssm.conv_step(dev, d[0], d[1], d[2], outs[0], state_out=outs[1], batch=rows, channels=channels,
                                 width=width, state_rows=rows, dtype=dtype, stream=stream)
        ferrum_gpu.ssm.scan_step(dev, d[0], d[0], d[3], d[4], d[4], d[5], outs[2], state_out=outs[3], groups=1,
                                 batch=rows, channels=channels, states=states, state_rows=rows, dtype=dtype,
                                 stream=stream)

    def results():
        return [o.copy_to_host(np.empty_like(v)) for o, v in zip(outs, (x, window, x, h))]

    with Capture(dev) as cap:  # the first calls of this type in the process
        calls(cap.stream)
    got = []
    for _ in range(3):
        cap.graph.launch()
        got.append(results())
        for o, v in zip(outs, (x, window, x, h)):
            o.copy_from_host(np.full_like(v, 7))
    calls(0)
    want = results()
    assert all(np.array_equal(p, q) for g in got for p, q in zip(g, want)), dtype
    assert all(not (v == 7).all() for v in want)
    print(dtype, "same", flush=True)
"""


def test_a_types_first_call_may_be_captured(gpu_device):
    """In a process of its own, whose first call of a type loads its code object."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrum-gpu_amd")
    ran = subprocess.run([sys.executable, "-c", FIRST_CALLS, root], capture_output=True, text=True, timeout=100)
    assert ran.returncode == 0, ran.stdout + ran.stderr
    assert ran.stdout.split() == ["float16", "same", "float32", "same"]
