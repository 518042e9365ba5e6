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
    built = programs.build(tmp_path_factory.mktemp("on_cpu"))

    def run(name, dtype, *args):
        got = subprocess.run([built[name, dtype], *map(str, args)], capture_output=True, text=True, timeout=300)
        assert got.returncode == 0, f"{name} {dtype} {args}: ended with {got.returncode}\n{got.stdout}{got.stderr}"

    return run


# Widths of every kernel of the norm, those that fill their team's threads and those that do not.
@pytest.mark.parametrize("dtype,rows,width", [
    ("bf16", 7, 8), ("bf16", 9, 64), ("bf16", 3, 512), ("bf16", 5, 1000), ("bf16", 9, 70), ("bf16", 5, 1088), ("bf16", 3, 1501),
    ("bf16", 4, 2560), ("bf16", 3, 4096), ("bf16", 3, 4099), ("bf16", 3, 5120), ("bf16", 2, 8200), ("bf16", 2, 16383),
    ("bf16", 2, 16400), ("bf16", 2, 17001), ("f32", 5, 1), ("f32", 7, 4), ("f32", 5, 260), ("f32", 5, 600), ("f32", 3, 1500),
    ("f32", 3, 4100), ("f32", 2, 8188), ("f32", 2, 9001)])
def test_norm_stays_within_its_arrays(program, dtype, rows, width):
    program("norm", dtype, rows, width)


@pytest.mark.parametrize("dtype,width", [("bf16", 200), ("bf16", 600), ("bf16", 2100), ("f32", 5000), ("bf16", 16400), ("f32", 601)])
def test_scales_of_rows_that_are_not_finite(program, dtype, width):
    program("norm", dtype, 6, width, "bad")


# 64 bits' definition at the sizes of one wave, one tile and several; offsets beyond the rows count as the nearest.
@pytest.mark.parametrize("args", [
    "f32 64 40 dense 1", "f32 61 700 dense 1", "bf16 66 300 dense 2", "bf16 64 1100 dense 1", "f32 1 1 dense 3", "f32 130 129 dense 2",
    "bf16 64 700 packed 0 300 300 310 700", "f32 37 200 packed -5 40 250 300", "f32 66 150 packed 3 10 10 140 145",
    "bf16 5 64 packed 0 1 2 3 4 5 6 64"])
def test_recurrence_stays_within_its_arrays(program, args):
    program("rec", *args.split())


# A search over offsets that fall could answer with a sequence behind the last one: where a wave then finds one's first
# or last token (as in the first three), it read or wrote a row behind the states' arrays.
@pytest.mark.parametrize("dtype,channels", [("bf16", 64), ("bf16", 7), ("f32", 64), ("f32", 13)])
@pytest.mark.parametrize("tokens,offsets", [
    (20, "0 20 5"), (20, "10 20 5"), (16, "0 16 5"), (16, "3 9 16 2"), (40, "9 5 40 1 1"), (700, "0 600 590 700 20"),
    (90, "-4 2 9 5 2147483647 1 1 1"), (700, "700 0 700 0")])
def test_falling_offsets_stay_within_the_arrays(program, dtype, channels, tokens, offsets):
    program("rec", dtype, channels, tokens, "packed", *offsets.split())


# Numbers of channel blocks and chains that the eight XCDs divide and others; launches from the first one on and
# around the one whose number passes the tags' 31 bits.
@pytest.mark.parametrize("blocks,chains", [(1, 1), (3, 1), (8, 1), (5, 8), (16, 3), (7, 7), (32, 1), (24, 2), (1, 13)])
@pytest.mark.parametrize("first", [0, 5, 2 ** 31 - 2])
def test_workgroups_share_the_tiles(program, blocks, chains, first):
    program("rec", "f32", blocks, chains, "places", first)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("channels,rows", [(64, 7), (37, 5), (1, 3), (260, 9)])
def test_one_token_is_a_sequence_of_one(program, dtype, channels, rows):
    program("rec", dtype, channels, 1, "step", rows)


# A wave, a tile of several waves, several tiles in and beyond one group of them.
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("channels,tokens,sequences", [(64, 20, 1), (64, 100, 1), (37, 128, 2), (64, 256, 1), (66, 600, 2),
                                                       (64, 1300, 1)])
def test_last_states_may_lie_over_first_ones(program, dtype, channels, tokens, sequences):
    program("rec", dtype, channels, tokens, "inplace", sequences)
