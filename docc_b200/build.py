"""Builds ``libdocc_b200_rt.so`` (the C-ABI runtime) for sm_100a with nvcc.

``python -m docc_b200.build`` compiles every ``csrc/*.cu`` into an object file (in
parallel) and links them into ``docc_b200/lib/libdocc_b200_rt.so``. The library has
no Python or torch dependency; the CUDA runtime is linked statically.

Where torch is installed, ``host/decode_calls.cpp`` is compiled beside it: the host side of
the shortest calls of ``docc_b200.ops`` for torch tensors, which reaches the library through
the addresses that ``ops`` binds and is not linked with it. It is built against the headers of
the installed torch and interpreter, and its file is named for both, so that one built for
others is never loaded. ``ops`` does without it; if it cannot be built, that is a warning.
"""
from __future__ import annotations

import glob
import hashlib
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor

_PKG = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_PKG)
CSRC = os.path.join(_PKG, "csrc")
INCLUDE = os.path.join(_ROOT, "include")
LIB_DIR = os.path.join(_PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libdocc_b200_rt.so")
HOST_SRC = os.path.join(_PKG, "host", "decode_calls.cpp")
HOST_NAME = "docc_b200_decode_calls"
_OBJ_DIR = os.path.join(_PKG, "build", "obj")
_STAMP = os.path.join(LIB_DIR, "libdocc_b200_rt.stamp")

NVCC_FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC",
    "-I" + INCLUDE, "-I" + CSRC,
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or add it to PATH")


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def source_hash() -> str:
    h = hashlib.sha256()
    files = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh", ".h"))]
    files.append(os.path.join(INCLUDE, "docc_b200", "rt.h"))
    for path in files:
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as fh:
            h.update(fh.read())
    h.update(" ".join(NVCC_FLAGS).replace(_ROOT, "").encode())
    return h.hexdigest()


def is_current() -> bool:
    if not (os.path.exists(LIB_PATH) and os.path.exists(_STAMP)):
        return False
    with open(_STAMP) as fh:
        return fh.read().strip() == source_hash()


def _torch_root():
    """The installed torch package's folder, without importing it; None if there is none."""
    spec = importlib.util.find_spec("torch")
    return spec.submodule_search_locations[0] if spec and spec.submodule_search_locations else None


def _torch_version() -> str:
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return "unknown"


def host_path():
    """Where the compiled host side for the installed torch and the running interpreter is; None without torch."""
    if _torch_root() is None:
        return None
    return os.path.join(LIB_DIR, f"{HOST_NAME}.{sysconfig.get_config_var('SOABI')}.torch-{_torch_version()}.so")


def _host_stamp() -> str:
    """What the compiled host side is made from; its stamp holds this."""
    h = hashlib.sha256(os.path.basename(host_path()).encode())
    for path in (HOST_SRC, os.path.join(INCLUDE, "docc_b200", "rt.h")):
        with open(path, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def host_is_current() -> bool:
    path = host_path()
    if path is None:
        return True
    try:
        with open(os.path.join(LIB_DIR, HOST_NAME + ".stamp")) as fh:
            return os.path.exists(path) and fh.read().strip() == _host_stamp()
    except FileNotFoundError:
        return False


def _build_host() -> None:
    path, torch = host_path(), _torch_root()
    if path is None:
        return
    for old in glob.glob(os.path.join(LIB_DIR, HOST_NAME + "*.so")):
        os.remove(old)
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", "-I" + INCLUDE,
           "-I" + os.path.join(torch, "include"), "-I" + os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], HOST_SRC, "-o", path, "-L" + os.path.join(torch, "lib"), "-lc10", "-ltorch_cpu",
           "-ltorch_python", "-ltorch"]
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
        failed = f"{res.stdout}\n{res.stderr}" if res.returncode != 0 else None
    except OSError as e:  # no such compiler
        failed = str(e)
    if failed is not None:
        warnings.warn(f"{os.path.basename(HOST_SRC)} could not be compiled; docc_b200.ops works without it, 4-13 us slower per call of a "
                      f"decoding step:\n{failed}", RuntimeWarning, stacklevel=3)
        return
    with open(os.path.join(LIB_DIR, HOST_NAME + ".stamp"), "w") as fh:
        fh.write(_host_stamp())


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile and link the runtime, and the compiled host side, where their sources changed since the last build."""
    if force or not is_current():
        _build_runtime(verbose)
    if force or not host_is_current():
        _build_host()
    return LIB_PATH


def _build_runtime(verbose: bool) -> None:
    nvcc = _nvcc()
    os.makedirs(_OBJ_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)

    def compile_one(src: str) -> str:
        obj = os.path.join(_OBJ_DIR, src[:-3] + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{res.stdout}\n{res.stderr}")
        if verbose:
            sys.stderr.write(res.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, _sources()))
    link = [nvcc, "-shared", "-o", LIB_PATH, *objs, "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "static"]
    res = subprocess.run(link, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    with open(_STAMP, "w") as fh:
        fh.write(source_hash())


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
