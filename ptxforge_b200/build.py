"""Build recipe for the sm_100a shared library ``libpf_b200.so`` (the C ABI of include/pf_b200.h).

    python -m ptxforge_b200.build            # builds in place, next to this file

nvcc cross-compiles for sm_100a on a machine without a GPU.  The CUDA runtime is linked
statically and the driver is reached through cudaGetDriverEntryPoint, so the library loads (and
reports PF_ENODEV) where no GPU driver is installed.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(HERE, "libpf_b200.so")
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    if os.path.exists(cand):
        return cand
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found: set CUDA_HOME")
    return found


# Translation units of the library, compiled side by side: the fused product's kernels and ABI, and the 8-bit operators'.
UNITS = ("pf_b200.cu", "ops8.cu")
OBJ_DIR = os.path.join(ROOT, "build")


def _includes(path: str, seen: set | None = None) -> set:
    """`path` and every header of this repository that it includes."""
    seen = set() if seen is None else seen
    if path in seen:
        return seen
    seen.add(path)
    with open(path) as f:
        names = re.findall(r'^\s*#include\s+"([^"]+)"', f.read(), re.M)
    for n in names:
        for d in (CSRC, INCLUDE):
            if os.path.exists(os.path.join(d, n)):
                _includes(os.path.join(d, n), seen)
    return seen


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd: list[str]) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    log = r.stdout + r.stderr
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + log[-6000:])
    return log


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile libpf_b200.so if any source is newer than it; return its path."""
    me = os.path.abspath(__file__)
    units = {u: os.path.join(CSRC, u) for u in UNITS}
    deps = {u: sorted(_includes(src)) + [me] for u, src in units.items()}
    if not force and not _stale(LIB, [d for ds in deps.values() for d in ds]):
        build_torch()
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs = {u: os.path.join(OBJ_DIR, u[:-3] + ".o") for u in UNITS}

    def compile_unit(u):
        log_path = objs[u] + ".ptxas.txt"
        if not force and os.path.exists(log_path) and not _stale(objs[u], deps[u]):
            with open(log_path) as f:
                return f.read()
        log = _run([nvcc_path(), *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "--expt-relaxed-constexpr",
                    "-Xcompiler", "-fPIC,-Wall", "-cudart", "static", "-I", INCLUDE, "-I", CSRC, "-Xptxas", "-v",
                    "-c", units[u], "-o", objs[u] + ".tmp"])
        with open(log_path, "w") as f:
            f.write(log)
        os.replace(objs[u] + ".tmp", objs[u])
        return log

    with ThreadPoolExecutor(len(UNITS)) as pool:
        log = "".join(pool.map(compile_unit, UNITS))
    _run([nvcc_path(), *ARCH_FLAGS, "-shared", "-cudart", "static", *objs.values(), "-o", LIB + ".tmp"])
    os.replace(LIB + ".tmp", LIB)
    with open(os.path.join(HERE, "libpf_b200.ptxas.txt"), "w") as f:
        f.write(log)
    if verbose:
        print(log)
    build_torch(force)
    return LIB


TORCH_SRC = os.path.join(CSRC, "torch_ops8.cpp")
TORCH_LIB = os.path.join(HERE, "_ops8.so")


def build_torch(force: bool = False) -> str | None:
    """Build _ops8.so, the 8-bit operators' torch side (a Python module over libpf_b200.so), where there are a torch with
    CUDA and a C++ compiler; the library itself needs neither."""
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError:
        return None
    cxx = shutil.which("g++")
    if torch.version.cuda is None or cxx is None:
        why = "this torch has no CUDA" if torch.version.cuda is None else "g++ not found"
        print(f"_ops8.so (the 8-bit operators on torch tensors) is not built: {why}", file=sys.stderr)
        return None
    # It fits one torch and one Python: another of either builds it again.
    built_for, stamp = f"{torch.__version__} {sysconfig.get_config_var('SOABI')}", os.path.join(OBJ_DIR, "ops8_torch.txt")
    same = False
    if os.path.exists(stamp):
        with open(stamp) as f:
            same = f.read() == built_for
    if force or not same or _stale(TORCH_LIB, sorted(_includes(TORCH_SRC)) + [os.path.abspath(__file__)]):
        cuda = os.path.dirname(os.path.dirname(nvcc_path()))
        include = [INCLUDE, *cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
        _run([cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", *(a for d in include for a in ("-isystem", d)), TORCH_SRC,
              "-o", TORCH_LIB + ".tmp", *(a for d in cpp_extension.library_paths() for a in ("-L", d)), "-lc10", "-lc10_cuda",
              "-ltorch_cpu", "-ltorch", "-ltorch_python", "-L", HERE, "-lpf_b200", "-Wl,-rpath,$ORIGIN"])
        os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
        os.makedirs(OBJ_DIR, exist_ok=True)
        with open(stamp, "w") as f:
            f.write(built_for)
    return TORCH_LIB


# The PTXForge source tree the runner plugs into: $PTXFORGE_REFERENCE, else a `reference` directory beside the
# repository.  Where neither exists the tuner CLI is not built (build_tune returns None).
REF_ROOT = os.environ.get("PTXFORGE_REFERENCE") or os.path.normpath(os.path.join(ROOT, os.pardir, "reference"))
TUNE_SRC = os.path.join(HERE, "host", "tune_b200.cpp")
TUNE_BIN = os.path.join(ROOT, "build", "ptxforge-tune-b200")


def tune_command(out: str, lib_dir: str, rpath: str, ref_root: str = REF_ROOT) -> list[str]:
    """g++ line for PTXForge's tuner CLI with the B200 runner, against the libpf_b200.so in lib_dir."""
    return ["g++", "-std=c++20", "-O2", "-Wall", "-Wextra", "-I", INCLUDE,
            "-I", os.path.join(ref_root, "core", "include"), "-I", os.path.join(ref_root, "compiler", "include"),
            TUNE_SRC, "-L", lib_dir, "-lpf_b200", f"-Wl,-rpath,{rpath}", "-lpthread", "-o", out]


def build_tune(force: bool = False, ref_root: str = REF_ROOT) -> str | None:
    """Build build/ptxforge-tune-b200 when the PTXForge headers are available (they are not shipped here:
    the runner is compiled inside the PTXForge tree it plugs into)."""
    if not os.path.isdir(os.path.join(ref_root, "core", "include", "ptxforge")):
        return None
    deps = [TUNE_SRC, LIB, os.path.join(INCLUDE, "ptxforge_b200", "b200_runner.hpp"), os.path.join(INCLUDE, "pf_b200.h")]
    if force or _stale(TUNE_BIN, deps):
        os.makedirs(os.path.dirname(TUNE_BIN), exist_ok=True)
        # $ORIGIN-relative rpath: the binary finds the library wherever the repository is copied
        cmd = tune_command(TUNE_BIN + ".tmp", HERE, "$ORIGIN/../ptxforge_b200", ref_root)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("g++ failed:\n" + (r.stdout + r.stderr)[-6000:])
        os.replace(TUNE_BIN + ".tmp", TUNE_BIN)
    return TUNE_BIN


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_tune(force="--force" in sys.argv))
