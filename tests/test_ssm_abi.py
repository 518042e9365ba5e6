"""The sequence filters' boundary without a GPU: the argument structs that the
Python package packs against the header's, the kernels that the host looks up
against those instantiated, and refusals that need no device."""

from __future__ import annotations

import ctypes
import itertools
import os
import re
import struct
import subprocess

import pytest

import ferrum_gpu
from ferrum_gpu import _native as N
from ferrum_gpu import ssm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "ferrum_gpu.h")
KERNELS = os.path.join(ROOT, "ferrum-gpu_amd", "csrc", "kernels")

PACKED = {"fg_conv_shape": ssm._shape_pack, "fg_scan_shape": ssm._scan_shape_pack,
          "fg_conv_forward_args": ssm._conv_forward_pack, "fg_conv_backward_args": ssm._conv_backward_pack,
          "fg_conv_step_args": ssm._conv_step_pack, "fg_scan_forward_args": ssm._scan_forward_pack,
          "fg_scan_backward_args": ssm._scan_backward_pack, "fg_scan_step_args": ssm._scan_step_pack}


def test_packed_structs_have_the_headers_sizes(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "ferrum_gpu.h"\nint main(void) {\n' +
                   "".join(f'  printf("{n} %zu\\n", sizeof({n}));\n' for n in PACKED) + "  return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True)
    sizes = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                         check=True).stdout.splitlines())
    for name, pack in PACKED.items():
        assert pack.__self__.size == int(sizes[name]), name


def _members(name):
    """Names of a struct's 8-byte members in order, those of fg_rows and fg_scan_inputs expanded."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    out = []
    for decl in body.split(";"):
        m = re.match(r"\s*(const\s+)?(\w+)\s+(.*)", decl, flags=re.S)
        if not m:
            continue
        for v in m.group(3).split(","):
            v = v.strip().lstrip("*")
            if m.group(2) == "fg_rows":
                out += [v, v + ".seq", v + ".row"]
            elif m.group(2) == "fg_scan_inputs":
                out += _members("fg_scan_inputs")
            else:
                out.append(v)
    return out


class _Recorder:
    """Stands in for the library: keeps the packed arguments."""

    def __getattr__(self, name):
        def call(handle, args, stream):
            self.args = args
            return 0
        return call


class _Device:
    ordinal, handle = 0, None


def _plan(cls, **fields):
    p = object.__new__(cls)
    p._setup(2, 8, None, 16, _Device(), "float32")
    p._p = ctypes.c_void_p(1)
    for k, v in fields.items():
        setattr(p, k, v)
    return p


def test_arguments_land_in_their_members(monkeypatch):
    """Every argument is given its own address; each has to reach the member of its name."""
    rec = _Recorder()
    monkeypatch.setattr(ssm, "_n", type("M", (), {"lib": rec, "check": staticmethod(N.check)}))
    as_member = {"A": "a", "B": "b", "C": "c", "D": "d", "grad_A": "grad_a", "grad_B": "grad_b", "grad_C": "grad_c",
                 "grad_D": "grad_d"}

    def check(struct_name, call, names):
        args = {n: 1000 * (i + 1) for i, n in enumerate(names)}
        call(**args)
        got = dict(zip(_members(struct_name), struct.unpack(f"={len(rec.args) // 8}q", rec.args)))
        for n, v in args.items():
            assert got[as_member.get(n, n)] == v, (struct_name, n)

    conv = _plan(ssm.ConvPlan, width=4, _state_shape=(2, 3, 16), _state_bytes=0)
    check("fg_conv_forward_args", conv.forward, ["x", "weight", "out", "bias", "initial", "final"])
    check("fg_conv_backward_args", conv.backward,
          ["x", "weight", "grad_out", "grad_x", "grad_weight", "grad_bias", "bias", "initial", "grad_initial",
           "grad_final"])
    scan = _plan(ssm.ScanPlan, states=4, groups=1, checkpoint_bytes=0)
    both = ["u", "delta", "A", "B", "C", "D", "z", "delta_bias"]
    check("fg_scan_forward_args", scan.forward, both + ["out", "initial", "final", "checkpoints"])
    check("fg_scan_backward_args", scan.backward,
          both + ["grad_out", "checkpoints", "grad_u", "grad_delta", "grad_A", "grad_B", "grad_C", "grad_D", "grad_z",
                  "grad_delta_bias", "grad_initial", "grad_final"])
    size = dict(batch=3, channels=16, state_rows=5, dtype="float16")
    check("fg_conv_step_args", lambda **k: ssm.conv_step(_Device(), **k, width=4, **size),
          ["x", "weight", "state", "out", "bias", "slots", "state_out"])
    check("fg_scan_step_args", lambda **k: ssm.scan_step(_Device(), **k, states=4, **size),
          both + ["state", "out", "slots", "state_out"])
    monkeypatch.undo()
    conv._p = scan._p = ctypes.c_void_p()


def test_every_kernel_that_the_host_looks_up_is_instantiated():
    """Names composed in ssm_ops.cpp against the code objects' symbols in the library."""
    blob = open(N.LIB_PATH, "rb").read()
    names = ["fg_scan_reduce_p", "fg_conv_reduce"]
    for t, most in (("f32", 4), ("bf16", 8), ("f16", 8)):
        for s, tail in itertools.product(("s1w1", "s2w1", "s4w1", "s4w2", "s4w4"), ("", "_any")):
            names += [f"fg_scan_{k}{t}_{s}{tail}" for k in ("", "local_", "back_", "back_local_")]
        names += [f"fg_scan_reduce_bc_{t}"]
        names += [f"fg_scan_step_{t}_l{n}{tail}" for n in (1, 2, 4, 8, 16) for tail in ("", "_any")]
        for w in range(2, ssm.MAX_WIDTH + 1):
            names += [f"fg_conv_{k}{t}_w{w}_v{n}" for k in ("", "step_")
                      for n in {1, 4, most if w <= 4 else 4}]
            names += [f"fg_conv_back_{t}_w{w}_v{n}" for n in (1, 4)]
    missing = [n for n in names if b"\0" + n.encode() + b"\0" not in blob]
    assert not missing, missing


def test_null_arguments_are_refused():
    lib = N.lib
    out = ctypes.c_void_p(5)
    for create in (lib.fg_conv_plan_create, lib.fg_scan_plan_create):
        assert create(None, b"", ctypes.byref(out)) == N.FG_ERR_INVALID_ARGUMENT and not out.value
    for call in (lib.fg_conv_forward, lib.fg_conv_backward, lib.fg_conv_step, lib.fg_scan_forward,
                 lib.fg_scan_backward, lib.fg_scan_step):
        assert call(None, b"", None) == N.FG_ERR_INVALID_ARGUMENT
        assert "is null" in N.last_error()
    assert lib.fg_scan_checkpoint_bytes(None, None) == N.FG_ERR_INVALID_ARGUMENT
    assert lib.fg_conv_plan_destroy(None) == N.FG_OK and lib.fg_scan_plan_destroy(None) == N.FG_OK


def test_types_and_activations_are_checked():
    for bad in ("float64", "int8", "bf16"):
        with pytest.raises(ValueError, match="dtype must be one of"):
            ssm._check_dtype(bad)
    with pytest.raises(ValueError, match="activation must be"):
        ssm._check_activation("gelu")


def test_tensors_are_checked_on_the_host():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 8, 16)
    rows = lambda v, **k: ssm._rows(v, (2, 8), 16, (2, 8), "float32", k.get("at", -1), "x")  # noqa: E731
    assert rows(x) == (x.data_ptr(), 128, 16)
    assert rows(torch.zeros(2, 8, 40)[..., 3:19])[1:] == (320, 40)
    assert rows(x[:1].expand(2, 8, 16))[1:] == (0, 16)
    assert rows(torch.zeros(2, 8, 2, 8))[1:] == (128, 16)
    for bad, why in ((x[:, :7], "shape"), (x.transpose(1, 2).contiguous().transpose(1, 2), "adjacent"),
                     (x.half(), "float16"), (torch.zeros(2, 8, 2, 16)[..., ::2], "adjacent"),
                     (torch.zeros(2, 8, 2, 9)[..., :8], "adjacent")):
        with pytest.raises(ValueError, match=why):
            rows(bad)
    with pytest.raises(ValueError, match="runs on GPU 0"):
        rows(x, at=0)
    flat = lambda v: ssm._flat(v, (4, 3), "float32", 48, -1, "w")  # noqa: E731
    assert flat(None) == 0
    for bad, why in ((torch.zeros(3, 4), "shape"), (torch.zeros(4, 3).double(), "float64"),
                     (torch.zeros(3, 4).t(), "contiguous")):
        with pytest.raises(ValueError, match=why):
            flat(bad)


@pytest.mark.parametrize("lead,width", [((2, 8), 16), ((8,), 16)])
def test_rows_without_their_last_axis_are_refused(lead, width):
    """A dense plan's (batch, length), a packed plan's (tokens), a step's (batch)."""
    torch = pytest.importorskip("torch")
    for bad in (torch.zeros(lead), torch.zeros(*lead, width, 1), torch.zeros(width)):
        with pytest.raises(ValueError, match="shape"):
            ssm._rows(bad, lead, width, (), "float32", -1, "x")
        with pytest.raises(ValueError, match="shape"):
            ssm._step_row(bad, (lead[0], width), (), "float32", -1, "x")


def test_package_exports_the_module():
    assert ferrum_gpu.ssm is ssm and "ssm" in ferrum_gpu.__all__


def test_streams_that_calls_take():
    """Handles, torch's streams (its default one has the handle 0), nothing of another GPU."""
    class Stream:
        def __init__(self, handle, index=0):
            self.cuda_stream, self.device_index = handle, index

    assert ssm._stream(0, 0) is None and ssm._stream(None, 0) is None and ssm._stream(77, 0) == 77
    assert ssm._stream(Stream(0), 0) == 1 and ssm._stream(Stream(5), 0) == 5
    with pytest.raises(ValueError, match="GPU 1"):
        ssm._stream(Stream(5, 1), 0)
    text = open(HEADER).read()
    assert re.search(r"#define FG_STREAM_NULL \(\(fg_stream_t\)1\)", text)


def test_a_tensor_without_a_gpu_says_why():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="runs on GPU 0; torch finds no GPU where this package was imported first"):
        ssm._rows(torch.zeros(2, 8, 16), (2, 8), 16, (), "float32", 0, "x")
