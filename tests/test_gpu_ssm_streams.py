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
