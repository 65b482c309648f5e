"""Build libcompactlogic_hip.so (gfx950) in-tree with hipcc, and the autograd extension over it.

Usage: ``python -m compactlogic_amd.build`` (or ``build()`` from Python).  Every source in
``csrc/*.hip`` is compiled to an object in ``_build/`` in parallel and linked into
``compactlogic_amd/libcompactlogic_hip.so``; ``csrc/autograd.cpp``, host code over torch's C++
interface, becomes ``compactlogic_amd/_autograd.so``.  The package loads these files only; nothing
is compiled at import time.
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
BUILD = PKG / "_build"
LIB = PKG / "libcompactlogic_hip.so"
AUTOGRAD = PKG / "_autograd.so"
ARCH = os.environ.get("CL_OFFLOAD_ARCH", "gfx950")

# -Xclang -target-feature -Xclang -packed-fp32-ops keeps the compiler from emitting packed
# fp32 arithmetic (v_pk_*_f32), which is avoided on these boxes.
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found; the HIP extension cannot be built")


def _compile(src: Path, hipcc: str) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [hipcc, *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src.name}:\n{proc.stdout}\n{proc.stderr}")
    return obj


def _run(cmd: list, what: str) -> None:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{proc.stdout}\n{proc.stderr}")


def _cxx() -> str:
    found = os.environ.get("CXX") or shutil.which("g++")
    if not found:
        raise RuntimeError("g++ not found; the autograd extension cannot be built")
    return found


def _compile_autograd() -> Path:
    from torch.utils.cpp_extension import include_paths
    obj = BUILD / "autograd.o"
    dirs = [*include_paths("cuda"), sysconfig.get_paths()["include"]]
    _run([_cxx(), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall",
          "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", "-DTORCH_EXTENSION_NAME=_autograd",
          *(a for d in dirs for a in ("-isystem", d)),
          "-c", str(CSRC / "autograd.cpp"), "-o", str(obj)], "autograd.cpp")
    return obj


def _link_autograd(obj: Path) -> None:
    import torch
    tmp = AUTOGRAD.with_suffix(".so.tmp")
    _run([_cxx(), "-shared", str(obj), "-o", str(tmp),
          f"-L{Path(torch.__file__).parent / 'lib'}", "-ltorch", "-ltorch_cpu", "-ltorch_python",
          "-lc10", "-lc10_hip", f"-L{PKG}", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"],
         "link of the autograd extension")
    os.replace(tmp, AUTOGRAD)


def build(verbose: bool = True) -> Path:
    """Compile every csrc/*.hip for gfx950 and link the shared library, then the autograd extension
    over it. Returns the library's path.  Where only the extension fails, this raises with the
    library in place."""
    hipcc = _hipcc()
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    workers = min(len(sources), max(1, (os.cpu_count() or 2) // 2), 8)
    with cf.ThreadPoolExecutor(max_workers=workers) as ex:
        autograd = ex.submit(_compile_autograd)
        objs = list(ex.map(lambda s: _compile(s, hipcc), sources))
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
        _run(cmd, "link")
        os.replace(tmp, LIB)
        try:
            _link_autograd(autograd.result())
        except Exception as e:
            # one of an earlier build goes with an earlier library
            AUTOGRAD.unlink(missing_ok=True)
            raise RuntimeError(f"built {LIB}, but not the autograd extension (the losses of "
                               f"policy.py and dropout need it): {e}") from e
    if verbose:
        print(f"built {LIB} from {len(sources)} sources", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    build()
