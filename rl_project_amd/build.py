"""Build libflsampler.so in-tree from ``rl_project_amd/csrc/*.hip`` for gfx950, and
the torch extension over it (``csrc/fl_autograd.cpp``).

    python -m rl_project_amd.build [-v]

Every ``.hip`` file is compiled by ``hipcc`` to an object (in parallel), then
linked into ``rl_project_amd/_lib/libflsampler.so``.  The library is a plain
C-ABI shared object (include/fl_sampler.h); Python loads it with ctypes.
"""

from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ_DIR = os.path.join(PKG, "_build")
LIB_DIR = os.path.join(PKG, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libflsampler.so")
AUTOGRAD_PATH = os.path.join(LIB_DIR, "_fl_autograd.so")
ARCH = os.environ.get("FL_OFFLOAD_ARCH", "gfx950")

# Correctly rounded float32 division (the reference's x / T is IEEE division),
# IEEE denormals (PyTorch's CPU kernels keep them), no packed-fp32 ops.  The
# scheduler's AMDGPU register-pressure trackers let the 16-bit row kernels
# keep their 64-VGPR row tile from the first read to the last use without
# spilling (the generic trackers misjudge the pressure and spill it).
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-fhip-fp32-correctly-rounded-divide-sqrt", "-fno-gpu-flush-denormals-to-zero",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-mllvm", "-amdgpu-use-amdgpu-trackers",
    "-mcode-object-version=5", "-Wall", "-Wno-unused-result",
]


# Per-file additions.  The float32 row kernel and the speculative verify are
# built for size: their latency-bound phases run long stretches of straight-line
# code once per row, and at -Os they measured faster on every float32
# workload (A/B on one box: uniform fp32 B=64 17.55 -> 16.90 us per launch,
# speculative step 177.3 -> 175.0 us, soft-capped Zipf 251.6 -> 247.2 us);
# the 16-bit row kernel measured slower at -Os and stays at -O3.
FILE_FLAGS = {"fl_rows32.hip": ["-Os"], "fl_spec.hip": ["-Os"]}


# The host-sanitizer build: AddressSanitizer and UndefinedBehaviorSanitizer on
# the host side only (every -fsanitize= behind -Xarch_host; the device code is
# built as usual, at -O1), linked against the shared sanitizer runtime, which
# the loading process must preload.  Only the C ABI's host code (argument
# checks, workspace sizing, launches) runs under it; no kernel is launched
# without a GPU.
SANITIZE_FLAGS = [
    "-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
    "-Xarch_host", "-fno-sanitize-recover=undefined", "-Xarch_host", "-fno-omit-frame-pointer", "-g",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: install ROCm or set HIPCC")


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, *FILE_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    if verbose and res.stderr.strip():
        print(res.stderr, flush=True)
    return obj


def _build_autograd(verbose: bool) -> str:
    """Compile and link csrc/fl_autograd.cpp (host code alone) against the installed torch."""
    import sysconfig

    import torch

    root = os.path.dirname(os.path.abspath(torch.__file__))
    tmp = AUTOGRAD_PATH + ".tmp"
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1",
           "-DUSE_ROCM=1", "-DTORCH_API_INCLUDE_EXTENSION_H", "-DTORCH_EXTENSION_NAME=_fl_autograd",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{p}" for p in (f"{root}/include", f"{root}/include/torch/csrc/api/include", "/opt/rocm/include",
                                      sysconfig.get_paths()["include"])),
           os.path.join(CSRC, "fl_autograd.cpp"), f"-L{root}/lib", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch",
           "-ltorch_python", "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"the autograd extension failed to build:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, AUTOGRAD_PATH)
    return AUTOGRAD_PATH


def build(verbose: bool = False, jobs: int = 0) -> str:
    """Compile every kernel source and link the shared library, and the autograd
    extension; returns the library's path."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    jobs = jobs or min(len(srcs), max(1, (os.cpu_count() or 2) // 2), 8)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        ext = ex.submit(_build_autograd, verbose)
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
        ext.result()
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def asan_runtime() -> str:
    """The shared AddressSanitizer runtime of ROCm's clang (to preload), or ''."""
    hits = sorted(glob.glob("/opt/rocm/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    return hits[-1] if hits else ""


def build_sanitized(out_dir: str, verbose: bool = False) -> str:
    """Build the library with the host sanitizers into ``out_dir``; returns its
    path.  Load it with FL_SAMPLER_LIB=<path> and the runtime from
    ``asan_runtime()`` in LD_PRELOAD."""
    os.makedirs(out_dir, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    flags = [f if f != "-O3" else "-O1" for f in HIPCC_FLAGS]
    jobs = min(len(srcs), max(1, (os.cpu_count() or 2) // 2), 8)

    def one(src):
        obj = os.path.join(out_dir, os.path.basename(src) + ".o")
        cmd = [hipcc(), *flags, *SANITIZE_FLAGS, "-c", src, "-o", obj]  # (-O1 throughout: no FILE_FLAGS)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"hipcc failed for {src}:\n{res.stdout}\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(one, srcs))
    out = os.path.join(out_dir, "libflsampler.so")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-Xarch_host", "-fsanitize=address",
           "-Xarch_host", "-fsanitize=undefined", "-shared-libsan", *objs, "-o", out]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    return out


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
