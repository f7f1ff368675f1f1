"""In-tree build of ``libapproxtorch_b200.so`` (hand-written CUDA for sm_100a, no torch headers) and of ``_binding.so``, the
native Python binding of the operators that are called where latency counts (torch headers, host code only).

    python -m approxtorch_b200.build [--force] [--verbose]

Each ``csrc/*.cu`` is compiled with ``nvcc -gencode arch=compute_100a,code=sm_100a`` into
``csrc/_obj/`` and linked into ``approxtorch_b200/lib/libapproxtorch_b200.so``, which the Python
side loads with ctypes; ``csrc/binding/binding.cpp`` is compiled by the host compiler and linked against that
library and torch's.  nvcc cross-compiles, so no GPU is needed to build.
"""

from __future__ import annotations

import concurrent.futures
import contextlib
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
SRC_DIR = os.path.join(PKG, "csrc")
OBJ_DIR = os.path.join(SRC_DIR, "_obj")
LIB_DIR = os.path.join(PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libapproxtorch_b200.so")
BINDING_SRC = os.path.join(SRC_DIR, "binding", "binding.cpp")
BINDING_PATH = os.path.join(LIB_DIR, "_binding.so")
HEADER = os.path.join(os.path.dirname(PKG), "include", "approxtorch_b200.h")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    if os.path.exists(cand):
        return cand
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build approxtorch_b200")
    return found


def _host_compiler_flags() -> list[str]:
    return ["-ccbin", "/usr/bin/g++"] if os.path.exists("/usr/bin/g++") else []


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(SRC_DIR, "*.cu")))


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile (if stale) and return the path of the shared library.

    Safe to call from several processes at once (every rank of a torchrun job imports the package): the
    build runs under an exclusive file lock, and the library is linked under a temporary name and moved into
    place atomically, so no process ever opens a half-written file."""
    with _build_lock():
        return _build_locked(force, verbose)


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compile (if stale) and return the path of the native binding; needs the library, torch and a host compiler."""
    with _build_lock():
        return _build_binding(force, verbose)


@contextlib.contextmanager
def _build_lock():
    import fcntl
    os.makedirs(LIB_DIR, exist_ok=True)
    with open(os.path.join(LIB_DIR, ".build.lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            yield
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)


def _build_locked(force: bool, verbose: bool) -> str:
    srcs = sources()
    headers = glob.glob(os.path.join(SRC_DIR, "*.cuh")) + [HEADER]
    os.makedirs(OBJ_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    nvcc = _nvcc()
    common = [nvcc, "-std=c++17", "-O3", "-lineinfo", *ARCH_FLAGS, *_host_compiler_flags(),
              "-Xcompiler", "-fPIC", "-Xptxas", "-v" if verbose else "-O3"]
    jobs = []
    for src in srcs:
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        if force or _stale(obj, [src] + headers):
            jobs.append((src, obj))

    def compile_one(job):
        src, obj = job
        proc = subprocess.run(common + ["-c", src, "-o", obj], capture_output=True, text=True)
        return src, proc

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as pool:
        for src, proc in pool.map(compile_one, jobs):
            if verbose or proc.returncode != 0:
                sys.stderr.write(f"--- {os.path.basename(src)}\n{proc.stdout}{proc.stderr}\n")
            if proc.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}")
    objs = [os.path.join(OBJ_DIR, os.path.basename(s)[:-3] + ".o") for s in srcs]
    if force or jobs or _stale(LIB_PATH, objs):
        tmp = f"{LIB_PATH}.{os.getpid()}.tmp"
        link = [nvcc, "-shared", *ARCH_FLAGS, *_host_compiler_flags(), "-o", tmp, *objs, "-lcudart"]
        proc = subprocess.run(link, capture_output=True, text=True)
        if proc.returncode != 0:
            sys.stderr.write(proc.stdout + proc.stderr)
            if os.path.exists(tmp):
                os.remove(tmp)
            raise RuntimeError("link of libapproxtorch_b200.so failed")
        os.replace(tmp, LIB_PATH)
    return LIB_PATH


def _build_binding(force: bool, verbose: bool) -> str:
    import importlib.util
    import sysconfig
    spec = importlib.util.find_spec("torch")
    if spec is None:
        raise RuntimeError("torch is not installed")
    torch_dir = os.path.dirname(spec.origin)
    if not force and not _stale(BINDING_PATH, [BINDING_SRC, HEADER, os.path.join(torch_dir, "version.py")]):
        return BINDING_PATH
    import torch
    abi = int(torch.compiled_with_cxx11_abi())
    include = os.path.join(torch_dir, "include")
    cuda_include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else shutil.which("g++") or "g++"
    tmp = f"{BINDING_PATH}.{os.getpid()}.tmp"
    cmd = [cxx, "-std=c++17", "-O2", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_binding",
           f"-D_GLIBCXX_USE_CXX11_ABI={abi}", "-isystem", include,
           "-isystem", os.path.join(include, "torch", "csrc", "api", "include"), "-isystem", sysconfig.get_paths()["include"],
           "-isystem", cuda_include, BINDING_SRC, "-o", tmp, "-L" + LIB_DIR, "-lapproxtorch_b200", "-Wl,-rpath,$ORIGIN",
           "-L" + os.path.join(torch_dir, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    try:
        proc = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as error:
        raise RuntimeError(f"{cxx}: {error}") from error
    if verbose or proc.returncode != 0:
        sys.stderr.write(f"--- binding.cpp\n{proc.stdout}{proc.stderr}\n")
    if proc.returncode != 0:
        if os.path.exists(tmp):
            os.remove(tmp)
        raise RuntimeError("build of _binding.so failed")
    os.replace(tmp, BINDING_PATH)
    return BINDING_PATH


if __name__ == "__main__":
    options = {"force": "--force" in sys.argv, "verbose": "--verbose" in sys.argv}
    print(build_library(**options))
    try:
        print(build_binding(**options))
    except RuntimeError as error:                            # the library serves everything else
        sys.stderr.write(f"{error}: no 8-bit floating point operators and no counter-based dropout from Python\n")
