"""The recurrence's, the norm's and dropout's boundary without a GPU: the argument
structs that the Python package packs against the header's, the kernels that the
host looks up against those instantiated, and refusals that need no device."""

from __future__ import annotations

import ctypes
import os
import re
import struct
import subprocess

import pytest

import ferrum_gpu
from ferrum_gpu import _native as N
from ferrum_gpu import norm, pointwise, ssm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "ferrum_gpu.h")

PACKED = {"fg_recurrence_shape": ssm._recurrence_shape_pack, "fg_recurrence_forward_args": ssm._recurrence_forward_pack,
          "fg_recurrence_backward_args": ssm._recurrence_backward_pack,
          "fg_recurrence_step_args": ssm._recurrence_step_pack, "fg_norm_shape": norm._shape_pack,
          "fg_norm_forward_args": norm._forward_pack, "fg_norm_backward_args": norm._backward_pack,
          "fg_dropout_args": pointwise._dropout_pack}


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
    """Names of a struct's 8-byte members in order, those of fg_rows and of inputs expanded."""
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
            elif m.group(2).endswith("_inputs"):
                out += _members(m.group(2))
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


def test_arguments_land_in_their_members(monkeypatch):
    """Every argument is given its own address; each has to reach the member of its name."""
    rec = _Recorder()
    library = type("M", (), {"lib": rec, "check": staticmethod(N.check)})
    for module in (ssm, norm, pointwise):
        monkeypatch.setattr(module, "_n", library)

    def check(struct_name, call, names, renamed={}, values={}):
        args = {n: 1000 * (i + 1) for i, n in enumerate(names)}
        call(**args, **values)
        members = _members(struct_name)
        got = dict(zip(members, struct.unpack(f"={len(rec.args) // 8}q", rec.args)))
        for n, v in {**args, **values}.items():
            v = struct.unpack("=q", struct.pack("=d", v))[0] if isinstance(v, float) else v
            assert got[renamed.get(n, n)] == v, (struct_name, n)

    plan = object.__new__(ssm.RecurrencePlan)
    plan._setup(2, 8, None, 16, _Device(), "float32")
    plan._p, plan.checkpoint_bytes = ctypes.c_void_p(1), 0
    both = ["x", "gate_a", "gate_x", "decay", "bias_a", "bias_x"]
    check("fg_recurrence_forward_args", plan.forward, both + ["out", "initial", "final", "checkpoints"])
    check("fg_recurrence_backward_args", plan.backward,
          both + ["grad_out", "checkpoints", "grad_x", "grad_gate_a", "grad_gate_x", "grad_decay", "grad_bias_a",
                  "grad_bias_x", "grad_initial", "grad_final"])
    check("fg_recurrence_step_args", lambda **k: ssm.recurrence_step(_Device(), **k, batch=3, channels=16, dtype="float16"),
          both + ["state", "out", "slots", "state_out"], values={"state_rows": 5, "rate": 3.5})

    rows = object.__new__(norm.NormPlan)
    rows.device, rows.rows, rows.width, rows.dtype, rows._groups, rows._at = _Device(), 4, 16, "float32", 1, 0
    rows._p = ctypes.c_void_p(1)
    values = {"rows": 3, "dropout": 0.25, "seed": 77, "offset": 88}
    check("fg_norm_forward_args", rows.forward, ["x", "out", "weight", "residual", "sum_out", "scales", "counter"],
          {"sum_out": "sum"}, values)
    check("fg_norm_backward_args", rows.backward,
          ["sum_in", "grad_out", "weight", "grad_sum", "grad_x", "grad_residual", "grad_weight", "counter"],
          {"sum_in": "sum"}, values)
    check("fg_dropout_args", lambda **k: pointwise.dropout(_Device(), **k, dtype="float32"), ["x", "out", "counter"],
          values={"n": 9, "p": 0.5, "seed": 3, "offset": 4})
    monkeypatch.undo()
    plan._p = rows._p = ctypes.c_void_p()


def test_every_kernel_that_the_host_looks_up_is_instantiated():
    """Names composed in rec_ops.cpp and norm_ops.cpp against the code objects' symbols in the library."""
    blob = open(N.LIB_PATH, "rb").read()
    names = ["fg_rec_reduce", "fg_norm_reduce"]
    for t in ("f32", "bf16", "f16"):
        names += [f"fg_rec_{k}{t}{p}{form}" for k in ("", "back_") for p in ("", "_packed")
                  for form in ("", "_stream", "_any")]
        names += [f"fg_rec_step_{t}_v{n}" for n in (1, 4)] + [f"fg_dropout_{t}"]
        names += [f"fg_norm_{k}{t}_c{c}_t{n}{form}" for k in ("", "back_") for form in ("", "_any")
                  for c, n in ((1, 64), (2, 64), (1, 256), (1, 512), (1, 1024), (2, 1024), (0, 1024))]
    missing = [n for n in names if b"\0" + n.encode() + b"\0" not in blob]
    assert not missing, missing


def test_null_arguments_are_refused():
    lib, out = N.lib, ctypes.c_void_p(5)
    for create in (lib.fg_recurrence_plan_create, lib.fg_norm_plan_create):
        assert create(None, b"", ctypes.byref(out)) == N.FG_ERR_INVALID_ARGUMENT and not out.value
    for call in (lib.fg_recurrence_forward, lib.fg_recurrence_backward, lib.fg_recurrence_step, lib.fg_norm_forward,
                 lib.fg_norm_backward, lib.fg_dropout):
        assert call(None, b"", None) == N.FG_ERR_INVALID_ARGUMENT
        assert "is null" in N.last_error()
    assert lib.fg_recurrence_checkpoint_bytes(None, None) == N.FG_ERR_INVALID_ARGUMENT
    assert lib.fg_recurrence_plan_destroy(None) == N.FG_OK and lib.fg_norm_plan_destroy(None) == N.FG_OK


def test_package_exports_the_modules():
    assert ferrum_gpu.norm is norm and "norm" in ferrum_gpu.__all__
    assert "RecurrencePlan" in ssm.__all__ and "dropout" in pointwise.__all__


def test_tensors_are_checked_on_the_host():
    torch = pytest.importorskip("torch")
    plan = object.__new__(norm.NormPlan)
    plan.device, plan.width, plan.dtype, plan._at = _Device(), 16, "bfloat16", 0
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    for bad, why in ((x[:3], "shape"), (x.float(), "float32"), (x.view(-1), "shape"), (x, "runs on GPU 0")):
        with pytest.raises(ValueError, match=why):
            plan._of(bad, 4, "x")
    for bad, why in ((x, "float8_e4m3fn"), (torch.zeros(4, 15, dtype=torch.uint8), "shape"),
                     (torch.zeros(4, 16, dtype=torch.uint8), "runs on GPU 0")):
        with pytest.raises(ValueError, match=why):
            plan._out8(bad, 4)


@pytest.mark.parametrize("places", [1, 2, 3, 7, 64, 672, 1000003, 2 ** 31 - 1, 2 ** 32 - 1])
def test_quotients_by_a_reciprocal(places):
    """The kernels' divisions: a product with (2^64 - 1) / d or (2^32 - 1) / d and one correction."""
    for n in (0, 1, places - 1, places, places + 1, 5 * places - 1, 2 ** 40, 2 ** 62 + 12345):
        q = n * ((2 ** 64 - 1) // places) >> 64
        rest = n - q * places
        assert 0 <= rest < 2 * places
    for n in (0, 1, places - 1, places, 2 ** 32 - 1):
        if n < 2 ** 32:
            q = n * ((2 ** 32 - 1) // places) >> 32
            assert 0 <= n - q * places < 2 * places
