"""Programs that run this package's kernels on the CPU: the kernels' headers, without their
statements of GPU assembly, built by ROCm's clang for the host against hip/hip_runtime.h of this folder."""

from __future__ import annotations

import os
import re
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
KERNELS = os.path.join(os.path.dirname(os.path.dirname(HERE)), "ferrum-gpu_amd", "csrc", "kernels")
CLANG = "/opt/rocm/llvm/bin/clang++"
_ASM = re.compile(r'\basm(?: volatile)?\((?:"[^"]*"|[^;"])*\);')


def build(to) -> dict:
    """Builds the programs of this folder in the folder `to`, one for each element type, all at a time.
    (program, type) -> the path of what can be run."""
    copies = os.path.join(str(to), "kernels")
    os.makedirs(copies, exist_ok=True)
    for name in os.listdir(KERNELS):
        if name.endswith((".hpp", ".h")):
            with open(os.path.join(KERNELS, name)) as f:
                text = f.read()
            with open(os.path.join(copies, name), "w") as f:
                f.write(_ASM.sub("", text).replace("__attribute__((address_space(4)))", ""))
    built = {(p, t): os.path.join(str(to), f"{p}_{t}") for p in ("rec", "norm") for t in ("f32", "bf16")}
    running = [subprocess.Popen([CLANG, "-std=c++17", "-O1", "-mf16c", "-w", f"-DTYPE={t.upper()}", "-I", HERE, "-I", copies,
                                 os.path.join(HERE, p + ".cpp"), "-o", exe]) for (p, t), exe in built.items()]
    for r in running:
        assert r.wait() == 0, r.args
    return built
