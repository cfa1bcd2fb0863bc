"""Builds the gfx950 HIP library libxgen_amd.so in-tree (hipcc, no torch headers) and the
torch operators' host library libxgen_amd_ops.so (g++, torch headers).

Each csrc/*.hip file is compiled to an object in parallel, then linked into
xgen_amd/_lib/libxgen_amd.so.  The library links libamdhip64.so.7; loaded after
`import torch`, it binds to the HIP runtime torch already loaded (same soname).
"""
from __future__ import annotations

import concurrent.futures
import os
import re
import shutil
import subprocess
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
INCLUDE = ROOT / "include"
OUT_DIR = PACKAGE / "_lib"
LIBRARY = OUT_DIR / "libxgen_amd.so"
OPERATORS = OUT_DIR / "libxgen_amd_ops.so"
OBJ_DIR = ROOT / "_build" / "xgen_amd"

ARCH = "gfx950"
HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-mcode-object-version=5",
    "-Wall",
    "-Wno-unused-function",
    # packed fp32 VALU forms are disabled for every kernel in this library
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]

# Sources whose asm statements hold values in accumulator registers by name, from one statement to the next.  The compiler
# is not aware of that: were it to use one of them itself (a spill), sums would be wrong without an error.
NAMED_ACCUMULATORS = frozenset({"mxfp4_gemm"})
_ACCUMULATOR = re.compile(r"(?<![\w.$@])a(?:\d+\b|\[)")


def hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(path).exists():
        raise RuntimeError("hipcc not found; the ROCm toolchain is required to build xgen_amd")
    return path


def _hipcc(src: Path, *args: str) -> None:
    cmd = [hipcc(), *HIP_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", str(src), *args]
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{proc.stdout}")


def foreign_accumulators(assembly: str) -> list[str]:
    """The instructions of gfx950 assembly, other than matrix products and reads of accumulators, that name an accumulator
    register, and those that use scratch memory."""
    found = []
    for line in assembly.splitlines():
        code = line.split(";")[0].strip()
        if not code or code.startswith(".") or code.endswith(":"):
            continue
        name, _, operands = code.partition(" ") if " " in code else code.partition("\t")
        if name.startswith("scratch_") or (_ACCUMULATOR.search(operands) and not name.startswith(("v_mfma_", "v_accvgpr_read"))):
            found.append(code)
    return found


def _check_accumulators(src: Path) -> None:
    """Raises if the compiler uses accumulator registers, or spills, in a source whose statements hold values in them."""
    assembly = OBJ_DIR / (src.stem + ".s")
    _hipcc(src, "--cuda-device-only", "-S", "-o", str(assembly))
    text = assembly.read_text()
    found = foreign_accumulators(text)
    if found or "v_mfma_" not in text:
        raise RuntimeError(f"{src.name}: the compiler uses accumulator registers or scratch that the kernels' statements "
                           f"hold values in: {found[:8]}")


def _compile(src: Path) -> Path:
    obj = OBJ_DIR / (src.stem + ".o")
    _hipcc(src, "-c", "-o", str(obj))
    if src.stem in NAMED_ACCUMULATORS:
        _check_accumulators(src)
    return obj


def _operators() -> Path:
    """csrc/torch_ops.cpp: host code only; links torch, and opens libxgen_amd.so at run time."""
    import torch
    root = Path(torch.__file__).resolve().parent
    rocm = Path(hipcc()).resolve().parent.parent
    tmp = OPERATORS.with_suffix(".so.tmp")
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1",
           "-DUSE_ROCM=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{INCLUDE}", "-isystem", str(root / "include"), "-isystem", str(root / "include/torch/csrc/api/include"),
           "-isystem", str(rocm / "include"), str(CSRC / "torch_ops.cpp"), "-o", str(tmp),
           f"-L{root / 'lib'}", "-ltorch_cpu", "-lc10", "-lc10_hip", "-ltorch_hip", "-ldl"]
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed for torch_ops.cpp:\n{proc.stdout}")
    os.replace(tmp, OPERATORS)
    return OPERATORS


def build(jobs: int | None = None, verbose: bool = False) -> Path:
    """Compiles every csrc/*.hip for gfx950 and links libxgen_amd.so (returns its path), and the
    torch operators' library beside it."""
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = jobs or min(len(sources), max(1, (os.cpu_count() or 4)))
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs + 1) as pool:
        operators = pool.submit(_operators)
        objects = list(pool.map(_compile, sources))
        operators.result()
    tmp = LIBRARY.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objects), "-o", str(tmp)]
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stdout}")
    os.replace(tmp, LIBRARY)
    if verbose:
        print(f"built {LIBRARY}")
        print(f"built {OPERATORS}")
    return LIBRARY


if __name__ == "__main__":
    build(verbose=True)
