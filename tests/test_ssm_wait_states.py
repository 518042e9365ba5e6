"""Wait states around the sequence filters' inline assembly, in the code objects
built from this tree: two instructions (or an s_nop that counts as two) between
a vector instruction that writes a register and a lane exchange that takes it, a
DPP operand or v_permlane32_swap.  The compiler keeps them for instructions of
its own, but sees nothing of what a statement of assembly writes."""

import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUILD = os.path.join(ROOT, "ferrum-gpu_amd", "csrc", "_build")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
NEEDED = 2


def _code_object(path):
    raw = open(path, "rb").read()
    if raw.startswith(b"__CLANG_OFFLOAD_BUNDLE__"):
        (n,), at = struct.unpack_from("<Q", raw, 24), 32
        for _ in range(n):
            off, size, name_len = struct.unpack_from("<3Q", raw, at)
            if b"gfx950" in raw[at + 24:at + 24 + name_len]:
                return raw[off:off + size]
            at += 24 + name_len
    return raw


def _registers(operand):
    """Numbers of the vector registers of one operand."""
    m = re.fullmatch(r"[-|]*v(\d+)\|?", operand) or re.fullmatch(r"[-|]*v\[(\d+):(\d+)\]\|?", operand)
    if not m:
        return ()
    return range(int(m[1]), int(m[m.lastindex]) + 1)


def _operands(line):
    """The instruction's name and its operands, modifiers not among them."""
    name, _, rest = line.partition(" ")
    return name, [x.split()[0] for x in rest.split(",") if x.strip()]


def _written(line):
    """Vector registers that a vector instruction writes."""
    name, ops = _operands(line)
    if not name.startswith("v_") or not ops:
        return set()
    return set(_registers(ops[0])) | (set(_registers(ops[1])) if "swap" in name else set())


def _exchanged(line):
    """Vector registers whose values an instruction takes from other lanes."""
    name, ops = _operands(line)
    if name.startswith("v_permlane"):
        return set(_registers(ops[0])) | set(_registers(ops[1]))
    if "_dpp" in name:
        return set(_registers(ops[1]))
    return set()


def _kernels(text):
    """Kernel -> its instructions [(address, line, branch target or None)]."""
    kernels, at = {}, None
    for line in text.splitlines():
        m = re.match(r"^([0-9a-f]+) <(\w+)>:", line)
        if m:
            base, at = int(m[1], 16), kernels.setdefault(m[2], [])
            continue
        m = re.match(r"^\s+(\S.*?)\s*// ([0-9A-F]+):.*?(?:<\w+?(?:\+0x([0-9a-f]+))?>)?$", line)
        if m and at is not None:
            branch = m[1].startswith(("s_branch", "s_cbranch"))
            at.append((int(m[2], 16), re.sub(r"\s+", " ", m[1]), base + int(m[3] or "0", 16) if branch else None))
    return kernels


def _missing(code):
    """Exchanges with fewer wait states behind a write of their registers, over
    every way that leads to them."""
    index = {a: i for i, (a, _, _) in enumerate(code)}
    before = [[] for _ in code]
    for i, (_, line, target) in enumerate(code):
        if target is not None:
            before[index[target]].append(i)
        if i + 1 < len(code) and not line.startswith(("s_branch", "s_endpgm")):
            before[i + 1].append(i)
    found = []

    def back(i, registers, states):
        for j in before[i]:
            line = code[j][1]
            if _written(line) & registers:
                return line
            n = re.match(r"s_nop (\d+)", line)
            more = states + (int(n[1]) + 1 if n else 1)
            if more < NEEDED:
                by = back(j, registers, more)
                if by:
                    return by
        return None

    for i, (_, line, _) in enumerate(code):
        registers = _exchanged(line)
        by = back(i, registers, 0) if registers else None
        if by:
            found.append((by, line))
    return found


def test_the_count_sees_what_is_missing():
    """Hand-written sequences: what is short, what is enough, and a way around a loop."""
    def code(*lines):
        return [(4 * i, *(x if isinstance(x, tuple) else (x, None))) for i, x in enumerate(lines)]

    swap, write = "v_permlane32_swap_b32_e32 v4, v5", "v_fmac_f32_dpp v5, v1, v2 row_newbcast:3 row_mask:0xf"
    assert _missing(code(write, "s_nop 0", swap)) == [(write, swap)]
    assert _missing(code(write, "v_exp_f32_e32 v9, v8", swap)) == [(write, swap)]
    assert not _missing(code(write, "s_nop 1", swap))
    assert not _missing(code(write, "s_nop 0", "ds_read_b32 v7, v8", swap))
    assert not _missing(code("v_mul_f32_e32 v6, v5, v4", swap))
    assert _missing(code("v_mov_b32_e32 v[4:5], v1", swap))
    dpp = "v_add_f32_dpp v1, v3, v5 quad_perm:[1,0,3,2] row_mask:0xf"
    assert _missing(code("v_mul_f32_e32 v3, v3, v3", dpp)) and not _missing(code("v_mul_f32_e32 v5, v3, v3", dpp))
    assert not _missing(code("v_cmp_lt_f32_e32 vcc, v4, v5", swap))
    loop = code(swap, "s_nop 3", write, ("s_cbranch_scc1 0", 0), "s_endpgm")
    assert _missing(loop) == [(write, swap)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_exchanges_wait_for_what_they_take(dtype, tmp_path):
    bundle = os.path.join(BUILD, f"ssm_{dtype}.hsaco")
    if not (os.path.exists(bundle) and os.path.exists(OBJDUMP)):
        pytest.skip("needs the built code object and llvm-objdump")
    path = tmp_path / "ssm.elf"
    path.write_bytes(_code_object(bundle))
    kernels = _kernels(subprocess.run([OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True).stdout)
    exchanges = sum(bool(_exchanged(line)) for code in kernels.values() for _, line, _ in code)
    assert len(kernels) > 60 and exchanges > 5000
    found = {k: v for k, v in ((k, _missing(code)) for k, code in kernels.items()) if v}
    assert not found, "\n".join(f"{k}: {len(v)}, first: {v[0][0]} -> {v[0][1]}" for k, v in found.items())
