"""The example block of the sequence filters: a prompt, the same tokens one by
one from a cache of slots, and its gradients."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_block(gpu_device):
    """In a process of its own, with torch's tensors on the GPU: torch finds
    none where the package was loaded before it.  float32: about 60 tokens of
    some ten roundings each leave 1e-4 at most; the slope's step of 1e-2 leaves
    its square and rounding of 1e-6 / 1e-2."""
    at = os.path.join(ROOT, "ferrum-gpu_amd", "examples", "sequence_filters.py")
    ran = subprocess.run([sys.executable, at], capture_output=True, text=True, timeout=100)
    assert ran.returncode == 0, ran.stderr
    got = dict(line.split(": ") for line in ran.stdout.splitlines())
    assert float(got["tokens against the whole"]) <= 1e-4
    assert float(got["same block forward"]) == 0.0
    assert float(got["slope against the gradient"]) <= 1e-2
