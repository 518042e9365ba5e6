"""The norm's, dropout's and the recurrence's kernels on the CPU (tests/on_cpu): their own code,
with arrays that end where nothing is mapped, so that an access behind one ends the program.
What a GPU would do with such an access depends on what lies behind the array."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "on_cpu"))
import programs  # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists(programs.CLANG), reason="needs ROCm's clang")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    built = {}

    def run(name, *args):
        if name not in built:
            built[name] = programs.build(name + ".cpp", tmp_path_factory.mktemp(name))
        got = subprocess.run([built[name], *map(str, args)], capture_output=True, text=True, timeout=300)
        assert got.returncode == 0, f"{name} {args}: ended with {got.returncode}\n{got.stdout}{got.stderr}"

    return run


# Widths of every kernel of the norm, those that fill their team's threads and those that do not.
@pytest.mark.parametrize("dtype,rows,width", [
    ("bf16", 7, 8), ("bf16", 9, 64), ("bf16", 3, 512), ("bf16", 5, 1000), ("bf16", 9, 70), ("bf16", 5, 1088), ("bf16", 3, 1501),
    ("bf16", 4, 2560), ("bf16", 3, 4096), ("bf16", 3, 4099), ("bf16", 3, 5120), ("bf16", 2, 8200), ("bf16", 2, 16383),
    ("bf16", 2, 16400), ("bf16", 2, 17001), ("f32", 5, 1), ("f32", 7, 4), ("f32", 5, 260), ("f32", 5, 600), ("f32", 3, 1500),
    ("f32", 3, 4100), ("f32", 2, 8188), ("f32", 2, 9001)])
def test_norm_stays_within_its_arrays(program, dtype, rows, width):
    program("norm", dtype, rows, width)
