"""Build librecap_b200.so in-tree with nvcc for sm_100a, and the compiled binding of its row
kernels (``_native.so``, C++ over torch) with the host compiler.

Usage: ``python -m recap_b200.build`` (or ``recap_b200.build.build()``).  Each is rebuilt
when a source it comes from, under ``recap_b200/csrc`` or ``include/``, is newer than it.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
REPO_DIR = PACKAGE_DIR.parent
CSRC = PACKAGE_DIR / "csrc"
INCLUDE = REPO_DIR / "include"
LIB_NAME = "librecap_b200.so"
LIB_PATH = PACKAGE_DIR / LIB_NAME
BUILD_DIR = PACKAGE_DIR / "_build"
BINDING = CSRC / "binding.cpp"
BINDING_PATH = PACKAGE_DIR / "_native.so"

SOURCES = ["layout.cu", "select.cu", "closure.cu", "cvk.cu", "coarse.cu", "fmha.cu", "refresh.cu", "selftest.cu",
           "exchange.cu", "rotate.cu", "norm.cu", "capi.cu"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    "--expt-relaxed-constexpr",
    "-Xptxas",
    "-v",
]


def _cuda_home() -> str:
    return os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _nvcc() -> str:
    cuda_home = _cuda_home()
    cand = Path(cuda_home) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found; set CUDA_HOME")
    return found


def _stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    inputs = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h"))
    inputs += list(INCLUDE.glob("*.h")) + [Path(__file__)]
    return any(p.stat().st_mtime > built for p in inputs)


def _binding_command() -> list[str]:
    """The compiler call of the binding, for the running Python and its torch."""
    import torch

    root = Path(torch.__file__).resolve().parent
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{root / 'include'}",
            f"-I{root / 'include/torch/csrc/api/include'}", f"-I{sysconfig.get_paths()['include']}",
            f"-I{Path(_cuda_home()) / 'include'}", str(BINDING), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
            "-ltorch_python"]


def _binding_stamp() -> str:
    """What a built binding belongs to, kept beside it: it loads into this Python and torch only."""
    import torch

    return f"python {sys.version_info[0]}.{sys.version_info[1]} {sysconfig.get_config_var('SOABI')}, torch {torch.__version__}\n"


def _binding_sources_newer() -> bool:
    inputs = [BINDING, INCLUDE / "recap_b200.h", Path(__file__)]
    return not BINDING_PATH.exists() or any(p.stat().st_mtime > BINDING_PATH.stat().st_mtime for p in inputs)


def _start_binding(force: bool) -> subprocess.Popen | None:
    """Start compiling the binding if it is out of date."""
    stamp = BINDING_PATH.with_suffix(".txt")
    if not force and not _binding_sources_newer() and stamp.exists() and stamp.read_text() == _binding_stamp():
        return None
    return subprocess.Popen([*_binding_command(), "-o", str(BINDING_PATH.with_suffix(".so.tmp"))], stdout=subprocess.PIPE,
                            stderr=subprocess.STDOUT, text=True)


def _finish_binding(process: subprocess.Popen | None) -> None:
    if process is None:
        return
    out, _ = process.communicate()
    if process.returncode != 0:
        raise RuntimeError(out)
    os.replace(BINDING_PATH.with_suffix(".so.tmp"), BINDING_PATH)
    BINDING_PATH.with_suffix(".txt").write_text(_binding_stamp())


def build(force: bool = False, verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile the binding and every kernel source and link the shared library; returns its path.
    The library needs nothing of the binding: where that does not compile (no host compiler, no headers of
    Python or torch), this says so on stderr, and the row kernels raise when they are called from Python."""
    binding, error = None, None
    try:
        binding = _start_binding(force)
    except (ImportError, OSError) as e:
        error = e
    try:
        path = _build_library(force, verbose)
    finally:
        try:
            _finish_binding(binding)
        except RuntimeError as e:
            error = e
    if error is not None:
        if _binding_sources_newer():
            BINDING_PATH.unlink(missing_ok=True)  # one of older sources would not fit the library
        print(f"the binding of the row kernels ({BINDING_PATH.name}) was not built; the library and all that does not call "
              f"them do without it: {error}", file=sys.stderr)
    return path


def _build_library(force: bool, verbose: bool) -> Path:
    if not force and not _stale():
        return LIB_PATH
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    objs = []
    procs = []
    for src in SOURCES:
        obj = BUILD_DIR / (Path(src).stem + ".o")
        objs.append(obj)
        cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-I", str(INCLUDE), "-c", str(CSRC / src), "-o", str(obj)]
        procs.append((src, cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    logs = []
    failed = []
    for src, cmd, p in procs:
        out, _ = p.communicate()
        logs.append(f"== {src}\n{out}")
        if p.returncode != 0:
            failed.append(src)
    (BUILD_DIR / "ptxas.log").write_text("\n".join(logs))
    if failed:
        raise RuntimeError("nvcc failed for " + ", ".join(failed) + "\n" + "\n".join(logs))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    link = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs), "-lcudart_static", "-ldl", "-lrt", "-lpthread"]
    r = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stdout)
    os.replace(tmp, LIB_PATH)
    if verbose:
        print("\n".join(logs))
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
