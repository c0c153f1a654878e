"""Build recipe for libghost_hip.so: hipcc for gfx950, one object per source, in-tree; and for
_lm_autograd.so, the Python extension (C++, torch's headers) around its language-model operators.

The library is a plain C-ABI shared object (include/ghost_hip.h); it depends only on the HIP
runtime.  At run time it binds to the libamdhip64.so.7 that torch has already loaded (the
package imports torch before loading the library), so torch streams and the kernels share
one HIP runtime.
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
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
LIBNAME = "libghost_hip.so"
EXTNAME = "_lm_autograd"
INCLUDE = PKG.parent / "include"
ARCH = "gfx950"

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    # Packed fp32 VALU ops are kept out of every kernel.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{INCLUDE}",
]


def hipcc() -> str:
    cand = os.environ.get("HIPCC") or shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(cand).exists() and shutil.which(cand) is None:
        raise RuntimeError("hipcc not found; set HIPCC or install ROCm")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


def library_path() -> Path:
    return LIBDIR / LIBNAME


def extension_path() -> Path:
    return LIBDIR / (EXTNAME + ".so")


def _run(cmd: list[str], what: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{res.stderr}")


def _torch_flags() -> tuple[list[str], list[str]]:
    """Compiler and linker flags of a Python extension over the installed torch."""
    import torch
    root = Path(torch.__path__[0])
    rocm = Path(shutil.which(hipcc()) or hipcc()).resolve().parent.parent
    compile_flags = [
        "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
        "-DTORCH_API_INCLUDE_EXTENSION_H",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f"-I{INCLUDE}", f"-isystem{root / 'include'}",
        f"-isystem{root / 'include/torch/csrc/api/include'}", f"-isystem{rocm / 'include'}",
        f"-isystem{sysconfig.get_paths()['include']}"]
    link_flags = [f"-L{root / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch",
                  "-ltorch_python"]
    return compile_flags, link_flags


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    """Compiles every csrc/*.hip for gfx950 and links libghost_hip.so, then the extension (always
    rebuilds)."""
    cc = hipcc()
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    srcs = sources()
    if not srcs:
        raise RuntimeError(f"no HIP sources under {CSRC}")

    def compile_one(src: Path) -> Path:
        obj = objdir / (src.stem + ".o")
        cmd = [cc, *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        errs = "\n".join(l for l in res.stderr.splitlines()
                         if "packed-fp32-ops" not in l)  # host pass does not know the feature
        if res.returncode != 0:
            raise RuntimeError(f"hipcc failed for {src.name}:\n{errs}")
        if verbose and errs.strip():
            print(errs, file=sys.stderr)
        return obj

    cxx = os.environ.get("CXX") or "g++"
    ext_compile, ext_link = _torch_flags()
    ext_obj = objdir / (EXTNAME + ".ext.o")

    n = jobs or min(len(srcs) + 1, max(1, min(8, os.cpu_count() or 1)))
    with cf.ThreadPoolExecutor(max_workers=n) as ex:
        ext = ex.submit(_run, [cxx, *ext_compile, "-c", str(CSRC / "lm_autograd.cpp"), "-o",
                               str(ext_obj)], "g++ for lm_autograd.cpp", verbose)
        objs = list(ex.map(compile_one, srcs))
        ext.result()
    out = library_path()
    tmp = out.with_suffix(".so.tmp")
    cmd = [cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, out)
    # next to libghost_hip.so, which it finds there
    ext_tmp = extension_path().with_suffix(".so.tmp")
    _run([cxx, "-shared", "-fPIC", str(ext_obj), "-o", str(ext_tmp), f"-L{LIBDIR}",
          f"-l:{LIBNAME}", *ext_link, "-Wl,-rpath,$ORIGIN"], "link of the extension", verbose)
    os.replace(ext_tmp, extension_path())
    return out


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
