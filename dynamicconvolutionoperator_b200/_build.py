"""Build ``libddpm_b200.so`` in-tree with nvcc for sm_100a.

Every ``csrc/*.cu`` file is compiled separately (in parallel, skipped when the
object is newer than the source and the shared headers) into ``_build/`` and
linked into ``dynamicconvolutionoperator_b200/libddpm_b200.so``. The library is
a plain C-ABI shared object (see ``include/ddpm_b200.h``); Python loads it with
ctypes, so no torch headers or torch ABI are involved.

``csrc/torch/*.cpp`` (the operators' autograd side, against torch's headers) goes
into ``_operators.so`` beside it, which links the library; another torch than the
one it was built with builds it again.

Usage: ``python -m dynamicconvolutionoperator_b200._build [--force] [--debug]``.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
INCLUDE = REPO_DIR / "include"
BUILD_DIR = REPO_DIR / "_build"
LIB_PATH = PKG_DIR / "libddpm_b200.so"
OPERATORS_PATH = PKG_DIR / "_operators.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
BASE_FLAGS = [
    "-std=c++17",
    "-O3",
    "-lineinfo",
    "--expt-relaxed-constexpr",
    "-Xcompiler",
    "-fPIC,-O3,-fvisibility=hidden",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or add CUDA's bin directory to PATH")
    return cand


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def _stale(obj: Path, src: Path, deps: list[Path]) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return any(p.stat().st_mtime > t for p in [src, *deps])


def _build_operators(force: bool, verbose: bool) -> None:
    """Compile and link ``_operators.so`` (needs the library)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = Path(_nvcc()).resolve().parents[1]
    includes = [*cpp_extension.include_paths(), str(cuda / "include"),
                sysconfig.get_paths()["include"]]
    flags = ["-std=c++17", "-O2", "-fPIC", "-fvisibility=hidden",
             "-DTORCH_EXTENSION_NAME=_operators", "-DTORCH_API_INCLUDE_EXTENSION_H",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             *(f"-isystem{p}" for p in includes)]

    def run(cmd: list[str], what: str) -> None:
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"{what} failed:\n{res.stdout}\n{res.stderr}")

    cxx = os.environ.get("CXX") or shutil.which("g++") or "g++"
    objs = []
    (BUILD_DIR / "torch").mkdir(parents=True, exist_ok=True)
    # the module fits the torch it was compiled against only: another one (or other
    # flags) has to compile it again, which no file's time shows
    stamp = BUILD_DIR / "torch" / "built_with"
    with_ = "\n".join([torch.__version__, sys.version, cxx, *flags])
    if not stamp.exists() or stamp.read_text() != with_:
        force = True
    for src in sorted((CSRC / "torch").glob("*.cpp")):
        obj = BUILD_DIR / "torch" / (src.stem + ".o")
        if force or _stale(obj, src, sorted(INCLUDE.glob("*.h"))):
            run([cxx, *flags, "-c", str(src), "-o", str(obj)], f"compiling {src.name}")
        objs.append(obj)
    if force or not OPERATORS_PATH.exists() or any(
        o.stat().st_mtime > OPERATORS_PATH.stat().st_mtime for o in objs
    ):
        tmp = OPERATORS_PATH.with_suffix(".so.tmp")
        libs = [f"-L{p}" for p in cpp_extension.library_paths()]
        # the shared C++ runtime by name: a second, static one (all that some images
        # have for linking) would not catch torch's exceptions, nor torch this one's
        run([cxx, "-shared", "-o", str(tmp), *map(str, objs), f"-L{PKG_DIR}", f"-l:{LIB_PATH.name}",
             *libs, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
             "-l:libstdc++.so.6", "-Wl,-rpath,$ORIGIN"], "linking _operators.so")
        os.replace(tmp, OPERATORS_PATH)
    stamp.write_text(with_)


def build(force: bool = False, debug: bool = False, verbose: bool = False) -> Path:
    """Compile and link the library; returns its path."""
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    if not sources:
        raise RuntimeError(f"no CUDA sources under {CSRC}")
    deps = _headers()
    extra = ["-DDDPM_CHECK_BOUNDS", "-G0"] if debug else []
    flags = ARCH_FLAGS + BASE_FLAGS + extra + [f"-I{INCLUDE}", f"-I{CSRC}"]

    def compile_one(src: Path) -> Path:
        obj = BUILD_DIR / (src.stem + ".o")
        if force or _stale(obj, src, deps):
            cmd = [nvcc, *flags, "-c", str(src), "-o", str(obj)]
            if verbose:
                print(" ".join(cmd), flush=True)
            res = subprocess.run(cmd, capture_output=True, text=True)
            if res.returncode != 0:
                raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
        return obj

    workers = min(len(sources), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(max_workers=workers) as pool:
        objs = list(pool.map(compile_one, sources))

    if force or not LIB_PATH.exists() or any(
        o.stat().st_mtime > LIB_PATH.stat().st_mtime for o in objs
    ):
        tmp = LIB_PATH.with_suffix(".so.tmp")
        cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs)]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB_PATH)
    _build_operators(force, verbose)
    return LIB_PATH


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--debug", action="store_true", help="device-side bounds checks")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args(argv)
    path = build(force=args.force, debug=args.debug, verbose=args.verbose)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
