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
