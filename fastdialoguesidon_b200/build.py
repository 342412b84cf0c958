"""Build recipe for the in-tree native library ``_lib/libfds_b200.so`` and the
Python extension ``_lib/_fds_torch.<python>-torch<version>.so``.

The library: nvcc, sm_100a only (``-gencode arch=compute_100a,code=sm_100a``),
static cudart, no torch headers: a plain C ABI (``include/fds_b200.h``) that any
FFI can load. The extension (``csrc/torch_shim.cpp``, g++, torch's headers)
checks the layer ops' tensors and calls that ABI. Both live inside the package
directory so that they travel with the source tree. ``python
fastdialoguesidon_b200/build.py`` builds the library where torch is not installed.
"""

from __future__ import annotations

import fcntl
import importlib.util
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from contextlib import contextmanager
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libfds_b200.so"
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
# ... and of the window kernel (csrc/window_kernel.cuh: 128 threads at 200, 128 at 56)
WINDOW_KERNEL_MARK = "window_tile_kernel"
WINDOW_LAUNCH_REGS = 128


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found (CUDA 12.8+ toolkit required to build the sm_100a library)")
    return cand


def extension_path() -> Path:
    """The extension of this Python and this torch: it is bound to the ABI of both, so another
    version's is another file."""
    import torch

    return LIB_DIR / f"_fds_torch.{sys.implementation.cache_tag}-torch{torch.__version__}.so"


def _newer(inputs: list[Path], output: Path) -> bool:
    """``output`` is missing, or older than one of ``inputs``."""
    return not output.exists() or any(f.stat().st_mtime > output.stat().st_mtime for f in inputs)


def _library_stale() -> bool:
    files = [CSRC / s for s in SOURCES]
    files += sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h"))
    files += sorted(INCLUDE_DIR.glob("*.h"))
    return _newer(files, LIB_PATH)


def _extension_stale() -> bool:
    return _has_torch() and _newer([CSRC / SHIM_SOURCE, *sorted(INCLUDE_DIR.glob("*.h"))], extension_path())


def _has_torch() -> bool:
    return importlib.util.find_spec("torch") is not None


def is_stale() -> bool:
    return _library_stale() or _extension_stale()


def _run(cmd: list[str], verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    return res.stdout + res.stderr


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library and the extension, each if a source of its own is newer
    (or ``force``). The library is in place whatever becomes of the extension, which
    a tree without torch has no use for. Processes that build at once do so in turn,
    and the later ones find what the first has built."""
    with ThreadPoolExecutor(max_workers=1) as pool:  # side by side
        extension = pool.submit(build_extension, force, verbose) if _has_torch() else None
        build_library(force, verbose)
        if extension is not None:
            extension.result()
    return LIB_PATH


@contextmanager
def _workspace(output: Path):
    """A directory of this process's own beside ``output``, while no other process
    builds ``output``."""
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    with open(LIB_DIR / f".{output.name}.lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        with tempfile.TemporaryDirectory(dir=LIB_DIR, prefix=".build-") as tmp:
            yield Path(tmp)


def build_library(force: bool = False, verbose: bool = False) -> Path:
    if not (force or _library_stale()):
        return LIB_PATH
    with _workspace(LIB_PATH) as work:
        if not (force or _library_stale()):  # built while this process waited
            return LIB_PATH
        # the sources compile side by side, each to an object, then link
        objs = [work / (Path(src).stem + ".o") for src in SOURCES]

        def compile_one(job: tuple[str, Path]) -> str:
            src, obj = job
            return _run([nvcc_path(), *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xptxas=-v", "-Xcompiler",
                         "-fPIC,-fvisibility=hidden", "-I", str(INCLUDE_DIR), "-c", "-o", str(obj), str(CSRC / src)], verbose)

        with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as pool:
            log = "".join(pool.map(compile_one, zip(SOURCES, objs)))
        linked = work / LIB_PATH.name
        _run([nvcc_path(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", str(linked), *map(str, objs)], verbose)
        if verbose:
            sys.stdout.write(log)
        check_launch_registers(log)
        os.replace(linked, LIB_PATH)
    return LIB_PATH


def build_extension(force: bool = False, verbose: bool = False) -> Path:
    path = extension_path()
    if not (force or _extension_stale()):
        return path
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parents[1]
    with _workspace(path) as work:
        if not (force or _extension_stale()):
            return path
        linked = work / path.name
        _run([shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
              "-I", str(INCLUDE_DIR), "-I", sysconfig.get_paths()["include"], "-isystem", str(root / "include"),
              "-isystem", str(root / "include/torch/csrc/api/include"), "-isystem", str(cuda / "include"),
              str(CSRC / SHIM_SOURCE), "-o", str(linked), "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10",
              "-lc10_cuda"], verbose)
        os.replace(linked, path)
    return path


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
