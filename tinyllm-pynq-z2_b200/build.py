"""Build the Q6W sm_100a shared library in-tree.

    python build.py            # -> q6w_b200/libq6w_b200.so

The library is plain nvcc output with an ``extern "C"`` ABI (see
include/q6w_b200.h); it links only the CUDA runtime, no torch.
"""

import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
SOURCES = ["csrc/codec.cu", "csrc/linear.cu", "csrc/model.cu", "csrc/paged.cu", "csrc/paged_decode.cu", "csrc/paged_tc.cu"]
OUT = HERE / "q6w_b200" / "libq6w_b200.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def nvcc():
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(path).exists():
        raise RuntimeError("nvcc not found")
    return path


# Kernels that divide their registers among warps (csrc/paged_tc.cu), by their part of
# the mangled name: a thread's number at launch, which the division needs exactly.
SPLIT_REGISTERS = {"5paged11rows_kernelI": 128}


def check_split_registers(log):
    """Raise if ptxas gave a kernel of SPLIT_REGISTERS another number of registers
    than its division needs (the library would refuse its calls)."""
    kernel = None
    for line in log.splitlines():
        entry = re.search(r"Compiling entry function '(\w+)'", line)
        if entry:
            kernel = entry.group(1)
        used = re.search(r"Used (\d+) registers", line)
        for name, need in SPLIT_REGISTERS.items():
            if used and kernel and name in kernel and int(used.group(1)) != need:
                raise RuntimeError(f"{kernel} was compiled to {used.group(1)} registers a thread, its warps divide {need}")


def build(verbose=False, jobs=None):
    inc = ["-I", str(ROOT / "include"), "-I", str(HERE / "csrc")]
    objs = []
    procs = []
    tmp = HERE / "_build"
    tmp.mkdir(exist_ok=True)
    for src in SOURCES:
        obj = tmp / (Path(src).stem + ".o")
        cmd = [nvcc(), *ARCH, *FLAGS, *inc, "-c", str(HERE / src), "-o", str(obj)]
        procs.append((src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    logs = []
    for src, obj, p in procs:
        out, _ = p.communicate()
        logs.append(f"== {src}\n{out}")
        if p.returncode != 0:
            sys.stderr.write(out)
            raise RuntimeError(f"nvcc failed on {src}")
        check_split_registers(out)
        objs.append(str(obj))
    link = [nvcc(), *ARCH, "-shared", "-o", str(OUT), *objs, "-lcudart"]
    subprocess.run(link, check=True)
    (tmp / "ptxas.log").write_text("\n".join(logs))
    if verbose:
        print("\n".join(logs))
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
