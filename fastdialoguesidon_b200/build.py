"""Build recipe for the in-tree native library ``_lib/libfds_b200.so`` and the
Python extension ``_lib/_fds_torch.so``.

The library: nvcc, sm_100a only (``-gencode arch=compute_100a,code=sm_100a``),
static cudart, no torch headers: a plain C ABI (``include/fds_b200.h``) that any
FFI can load. The extension (``csrc/torch_shim.cpp``, g++, torch's headers)
checks the layer ops' tensors and calls that ABI. Both live inside the package
directory so that they travel with the source tree.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libfds_b200.so"
SHIM_PATH = LIB_DIR / "_fds_torch.so"
INCLUDE_DIR = REPO_DIR / "include"

SHIM_SOURCE = "torch_shim.cpp"
SOURCES = ["fds_capi.cu", "fds_rope_static.cu", "fds_int8.cu", "fds_norm.cu", "fds_window.cu"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]

# The attention kernels split their register file with setmaxnreg
# (csrc/attn_kernel.cuh RegSplit: 2 x 128 softmax threads at 224 or 208, 128
# control threads at 56 or 88). That
# split assumes the CTA is launched with exactly this many registers per
# thread; a different count could make the increase wait forever, so the build
# refuses to produce a library in that case.
ATTN_KERNEL_MARK = "attn_fwd_kernel"
ATTN_LAUNCH_REGS = 168
# ... and of the window kernel (csrc/window_kernel.cuh: 128 threads at 208, 128 at 48)
WINDOW_KERNEL_MARK = "window_tile_kernel"
WINDOW_LAUNCH_REGS = 128


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found (CUDA 12.8+ toolkit required to build the sm_100a library)")
    return cand


def _inputs() -> list[Path]:
    files = [CSRC / s for s in (*SOURCES, SHIM_SOURCE)]
    files += sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h"))
    files += sorted(INCLUDE_DIR.glob("*.h"))
    return files


def is_stale() -> bool:
    if not (LIB_PATH.exists() and SHIM_PATH.exists()):
        return True
    mtime = min(LIB_PATH.stat().st_mtime, SHIM_PATH.stat().st_mtime)
    return any(f.stat().st_mtime > mtime for f in _inputs())


def _run(cmd: list[str], verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    return res.stdout + res.stderr


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library and the extension if any source is newer (or ``force``)."""
    if not force and not is_stale():
        return LIB_PATH
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    # the sources compile side by side, each to an object, then link
    objs = [LIB_DIR / (Path(src).stem + ".o") for src in SOURCES]

    def compile_one(job: tuple[str, Path]) -> str:
        src, obj = job
        return _run([nvcc_path(), *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xptxas=-v", "-Xcompiler",
                     "-fPIC,-fvisibility=hidden", "-I", str(INCLUDE_DIR), "-c", "-o", str(obj), str(CSRC / src)], verbose)

    with ThreadPoolExecutor(max_workers=min(len(SOURCES) + 1, os.cpu_count() or 1)) as pool:
        shim = pool.submit(_build_shim, verbose)
        log = "".join(pool.map(compile_one, zip(SOURCES, objs)))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    _run([nvcc_path(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", str(tmp), *map(str, objs)], verbose)
    for obj in objs:
        obj.unlink()
    shim.result()
    if verbose:
        sys.stdout.write(log)
    check_launch_registers(log)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def _build_shim(verbose: bool) -> None:
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parents[1]
    tmp = SHIM_PATH.with_suffix(".so.tmp")
    _run([shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          "-I", str(INCLUDE_DIR), "-I", sysconfig.get_paths()["include"], "-isystem", str(root / "include"),
          "-isystem", str(root / "include/torch/csrc/api/include"), "-isystem", str(cuda / "include"),
          str(CSRC / SHIM_SOURCE), "-o", str(tmp), "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10",
          "-lc10_cuda"], verbose)
    os.replace(tmp, SHIM_PATH)


def check_launch_registers(ptxas_log: str) -> None:
    """Every kernel that splits its registers must launch with the count its split assumes."""
    for mark, expected in ((ATTN_KERNEL_MARK, ATTN_LAUNCH_REGS), (WINDOW_KERNEL_MARK, WINDOW_LAUNCH_REGS)):
        current, seen = None, 0
        for line in ptxas_log.splitlines():
            if "Compiling entry function" in line:
                current = line
            elif current and "Used" in line and "registers" in line:
                if mark in current:
                    regs = int(line.split("Used")[1].split("registers")[0])
                    if regs != expected:
                        raise RuntimeError(f"attention kernel launches with {regs} registers per thread, expected "
                                           f"{expected} (the setmaxnreg split depends on it): {current}")
                    seen += 1
                current = None
        if seen == 0:
            raise RuntimeError(f"no {mark} found in the ptxas report")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
