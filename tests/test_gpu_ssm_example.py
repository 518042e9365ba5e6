"""The example block of the sequence filters: a prompt, the same tokens one by
one from a cache of slots, and its gradients."""

from __future__ import annotations

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_block(gpu_device):
    """float32: about 60 tokens of some ten roundings each leave 1e-4 at most;
    the slope's step of 1e-2 leaves its square and rounding of 1e-6 / 1e-2."""
    at = os.path.join(ROOT, "ferrum-gpu_amd", "examples", "sequence_filters.py")
    spec = importlib.util.spec_from_file_location("sequence_filters", at)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    torch.manual_seed(0)
    got = module.main(gpu_device)
    assert got["tokens against the whole"] <= 1e-4
    assert got["same block forward"] == 0.0
    assert got["slope against the gradient"] <= 1e-2
