"""Build libfpemu.so (the C-ABI library) in-tree for sm_100a.

    python fp-emulation_b200/build.py [--force] [--verbose]

Every ``csrc/*.cu`` is one translation unit (the kernel headers are included
there); they are compiled side by side by nvcc for ``-gencode
arch=compute_100a,code=sm_100a``, each again only when it or a header changed,
and linked with the static CUDA runtime, so the library only needs the driver at
run time.  The output lands next to the Python package that loads it
(``fp_emulation/libfpemu.so``).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
OUT = HERE / "fp_emulation" / "libfpemu.so"

NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC,-O2",
    "--expt-relaxed-constexpr",
]
OBJ = HERE / "build"


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + \
        sorted(INCLUDE.glob("*.h"))


def up_to_date() -> bool:
    if not OUT.exists():
        return False
    t = OUT.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in sources())


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return OUT
    OBJ.mkdir(exist_ok=True)
    headers = max(p.stat().st_mtime for p in sources() + [Path(__file__)] if p.suffix != ".cu")

    def compile_one(src):
        obj = OBJ / (src.stem + ".o")
        if not force and not verbose and obj.exists() and obj.stat().st_mtime > max(src.stat().st_mtime, headers):
            return obj, None
        cmd = [nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + \
            [f"-I{INCLUDE}", "-c", str(src), "-o", str(obj) + ".tmp.o"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode == 0:
            os.replace(str(obj) + ".tmp.o", obj)
        return obj, res

    units = sorted(CSRC.glob("*.cu"))
    with ThreadPoolExecutor(len(units)) as pool:
        done = list(pool.map(compile_one, units))
    for obj, res in done:
        if res is not None and (verbose or res.returncode != 0):
            sys.stderr.write(res.stdout + res.stderr)
        if res is not None and res.returncode != 0:
            raise RuntimeError(f"nvcc failed ({res.returncode}) on {obj.stem}.cu")
    link = subprocess.run([nvcc(), "-shared", "-cudart", "static", "-gencode", "arch=compute_100a,code=sm_100a"]
                          + [str(obj) for obj, _ in done] + ["-o", str(OUT) + ".tmp"], capture_output=True, text=True)
    if link.returncode != 0:
        sys.stderr.write(link.stdout + link.stderr)
        raise RuntimeError(f"linking failed ({link.returncode})")
    os.replace(str(OUT) + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
