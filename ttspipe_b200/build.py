"""Build ``libnf4b200.so`` in-tree with nvcc for sm_100a.

Each ``csrc/*.cu`` is compiled separately (in parallel) with
``-gencode arch=compute_100a,code=sm_100a`` and linked into one shared library
next to this file, so it travels with the source tree. The CUDA runtime is
linked statically: the library carries its own runtime and shares only the
driver (and therefore the current context and streams) with the PyTorch that
calls it. ``csrc/pagedkv_bind.cpp`` then becomes ``_pagedkv.so`` beside it, a Python
module against this PyTorch's headers; the library needs neither it nor PyTorch.
``python -m ttspipe_b200.build`` rebuilds when a source is newer than what was built
from it, and the binding also for another PyTorch, Python or compiler.
"""

from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = PKG / "_build"
LIB = PKG / "libnf4b200.so"
BIND = PKG / "_pagedkv.so"
BIND_SRC = CSRC / "pagedkv_bind.cpp"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr",
              "-Xptxas", "-O3"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise FileNotFoundError("nvcc not found (set NVCC or install CUDA 12.9)")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def up_to_date() -> bool:
    if not LIB.exists():
        return False
    t = LIB.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in _deps())


def _cxx_runtime() -> list[str]:
    """The C++ runtime that this process's PyTorch runs on, to link the binding against. A compiler that has only
    the static one would put a second copy into the binding; two of them in a process crash where one formats numbers
    with the other's locale, as every refusal that names a shape does."""
    with open("/proc/self/maps") as maps:
        found = {line.split()[-1] for line in maps if "/libstdc++.so" in line}
    return sorted(found)


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile the Python binding of the paged KV cache. Returns its path."""
    cxx = os.environ.get("CXX") or shutil.which("g++")
    deps, stamp = [BIND_SRC, *INCLUDE.glob("*.h")], BUILD / "pagedkv_bind.txt"
    made_for = f"{importlib.metadata.version('torch')} {sys.version} {cxx}"
    if (not force and BIND.exists() and all(p.stat().st_mtime <= BIND.stat().st_mtime for p in deps)
            and stamp.exists() and (not cxx or stamp.read_text() == made_for)):
        return BIND
    if not cxx:
        raise FileNotFoundError("no C++ compiler (set CXX or install g++)")
    import sysconfig

    import torch

    BUILD.mkdir(exist_ok=True)
    home = Path(torch.__file__).resolve().parent
    inc = [INCLUDE, home / "include", home / "include" / "torch" / "csrc" / "api" / "include",
           sysconfig.get_paths()["include"]]
    tmp = BIND.with_suffix(".so.tmp")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{i}" for i in inc), str(BIND_SRC),
           f"-L{home / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10", *_cxx_runtime(), "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True, env=dict(os.environ, TMPDIR=str(BUILD)))
    if r.returncode != 0:
        raise RuntimeError(f"{cxx} failed on {BIND_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BIND)
    stamp.write_text(made_for)
    return BIND


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    """Compile every kernel source and link the shared library, then the binding (not where there is no PyTorch).
    Returns the library's path."""
    build_library(force=force, verbose=verbose, ptxas_info=ptxas_info)
    if importlib.util.find_spec("torch") is None:
        print("no PyTorch: the paged cache's Python binding is left out", file=sys.stderr)
    else:
        build_binding(force=force, verbose=verbose)
    return LIB


def build_library(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    """Compile every kernel source and link the shared library. Returns its path."""
    if not force and up_to_date() and not ptxas_info:
        return LIB
    BUILD.mkdir(exist_ok=True)
    cc = nvcc()
    extra = ["-Xptxas", "-v"] if ptxas_info else []
    env = dict(os.environ, TMPDIR=str(BUILD))  # nvcc's intermediate files stay in the build folder

    def compile_one(src: Path) -> tuple[Path, str]:
        obj = BUILD / (src.stem + ".o")
        cmd = [cc, *ARCH, *NVCC_FLAGS, *extra, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True, env=env)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        return obj, r.stderr

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, sources()))
    if ptxas_info:
        for _, err in results:
            sys.stdout.write(err)
    objs = [str(o) for o, _ in results]
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *objs]
    r = subprocess.run(cmd, capture_output=True, text=True, env=env)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv,
                ptxas_info="--ptxas" in sys.argv))
