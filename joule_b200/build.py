"""Build the CUDA library in-tree: joule_b200/libjoule_moe.so (sm_100a).

    python -m joule_b200.build            # incremental
    python -m joule_b200.build --force    # rebuild everything

Each .cu under csrc/ compiles to an object in parallel; the objects link into
one shared library with a static CUDA runtime. No torch headers are used:
the library's ABI is plain C (include/joule_moe.h). csrc/kv4_call.c, which
needs Python's headers alone, becomes joule_b200/_kv4_call with this interpreter's
suffix (another one does not load it, and goes without).
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = PKG / "_build"
LIB = PKG / "libjoule_moe.so"
CALL = PKG / f"_kv4_call{sysconfig.get_config_var('EXT_SUFFIX')}"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I", str(ROOT / "include"), "-I", str(CSRC)]


def nvcc() -> str:
    cand = [os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"]
    for c in cand:
        if c and Path(c).exists():
            return c
    raise RuntimeError("nvcc not found")


def _compile(src: Path, force: bool, extra: list[str]) -> Path:
    obj = OBJ / (src.stem + ".o")
    deps = [src] + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted((ROOT / "include").glob("*.h"))
    if not force and obj.exists() and obj.stat().st_mtime >= max(d.stat().st_mtime for d in deps):
        return obj
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stderr}")
    if os.environ.get("JL_PTXAS_VERBOSE"):
        sys.stderr.write(r.stderr)
    return obj


def _call_module(force: bool) -> None:
    src = CSRC / "kv4_call.c"
    deps = [src, ROOT / "include" / "joule_moe.h"]
    (PKG / "_kv4_call.so").unlink(missing_ok=True)  # one without a suffix would be loaded by any interpreter
    if not force and CALL.exists() and CALL.stat().st_mtime >= max(d.stat().st_mtime for d in deps):
        return
    cc = os.environ.get("CC") or shutil.which("gcc") or shutil.which("cc")
    if not cc:
        raise RuntimeError("no C compiler")
    cmd = [cc, "-O2", "-shared", "-fPIC", "-I", sysconfig.get_paths()["include"], "-I", str(ROOT / "include"), str(src),
           "-o", str(CALL), "-lm"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cc} failed for {src.name}:\n{r.stderr}")


def build(force: bool = False, verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    extra = ["-Xptxas", "-v"] if verbose else []
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, extra), srcs))
    if force or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs), "-lcuda"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    _call_module(force)
    return LIB


if __name__ == "__main__":
    if "-v" in sys.argv:
        os.environ["JL_PTXAS_VERBOSE"] = "1"
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
