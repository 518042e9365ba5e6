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


def build(program: str, to) -> str:
    """Builds `program` (.cpp, of this folder) in the folder `to`; the path of what can be run."""
    copies = os.path.join(str(to), "kernels")
    os.makedirs(copies, exist_ok=True)
    for name in os.listdir(KERNELS):
        if name.endswith((".hpp", ".h")):
            with open(os.path.join(KERNELS, name)) as f:
                text = f.read()
            with open(os.path.join(copies, name), "w") as f:
                f.write(_ASM.sub("", text).replace("__attribute__((address_space(4)))", ""))
    exe = os.path.join(str(to), program.removesuffix(".cpp"))
    subprocess.run([CLANG, "-std=c++17", "-O1", "-mf16c", "-Wno-everything", "-I", HERE, "-I", copies,
                    os.path.join(HERE, program), "-o", exe], check=True)
    return exe
