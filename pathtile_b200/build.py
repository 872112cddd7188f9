"""Build ``pathtile_b200/libpathtile_b200.so`` (sm_100a) in-tree with nvcc.

Every ``.cu`` unit under ``pathtile_b200/csrc`` is compiled in parallel for
``-gencode arch=compute_100a,code=sm_100a`` and linked into one shared library
with a static CUDA runtime, so the file is self-contained apart from the
driver.  Rebuilds only when a source or header is newer than the library.

``csrc/binding/sequence.cpp``, the sequence operators' binding to torch, becomes
the extension module ``pathtile_b200/_sequence.so`` beside it (g++, linked
against torch and the library).

Usage: ``python -m pathtile_b200.build [--force] [--verbose-ptxas]``.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libpathtile_b200.so"
BINDING_SRC = CSRC / "binding" / "sequence.cpp"
BINDING = PKG / "_sequence.so"
OBJ_DIR = ROOT / "_build" / "obj"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA 12.9 toolkit is required to build pathtile_b200")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in _deps())


def binding_needs_build() -> bool:
    if not BINDING.exists():
        return True
    t = BINDING.stat().st_mtime
    return any(p.stat().st_mtime > t for p in [BINDING_SRC, *INCLUDE.glob("*.h")])


def build_binding(force: bool = False) -> Path:
    """Compile the torch binding of the sequence operators; the library has to be there."""
    if not force and not binding_needs_build():
        return BINDING
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    # The system's compiler, which nvcc uses too: one that brings parts of its own C++ library
    # would put a second copy of them beside torch's.
    cxx = shutil.which("g++") or "g++"
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
           *(f"-isystem{p}" for p in include_paths("cuda")), f"-I{sysconfig.get_paths()['include']}",
           str(BINDING_SRC), "-o", str(tmp), *(f"-L{p}" for p in library_paths()),
           "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
           f"-L{PKG}", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {BINDING_SRC.name}:\n{res.stderr}\n{res.stdout}")
    os.replace(tmp, BINDING)
    return BINDING


def _compile(src: Path, verbose_ptxas: bool) -> tuple[Path, str]:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [nvcc_path(), *ARCH_FLAGS, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o", str(obj)]
    if verbose_ptxas:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stderr}\n{res.stdout}")
    return obj, res.stderr


def build(force: bool = False, verbose_ptxas: bool = False, jobs: int | None = None) -> Path:
    """Compile and link the library and its torch binding; returns the library's path."""
    if not force and not verbose_ptxas and not needs_build():
        build_binding()
        return LIB
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    srcs = sources()
    jobs = jobs or max(1, min(len(srcs), os.cpu_count() or 1))
    logs: list[str] = []
    objs: list[Path] = []
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        for obj, log in ex.map(lambda s: _compile(s, verbose_ptxas), srcs):
            objs.append(obj)
            if log.strip():
                logs.append(log)
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc_path(), *ARCH_FLAGS, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}\n{res.stdout}")
    os.replace(tmp, LIB)
    build_binding(force)
    if verbose_ptxas:
        sys.stderr.write("\n".join(logs))
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose-ptxas", action="store_true", help="print ptxas register/smem usage")
    args = ap.parse_args()
    path = build(force=args.force, verbose_ptxas=args.verbose_ptxas)
    print(path)


if __name__ == "__main__":
    main()
