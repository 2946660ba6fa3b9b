"""Builds libfp4x.so (the HIP kernels and their C ABI) and _fp4x_host.so (the
compiled host side of some eager calls) in-tree for gfx950.

    python build.py            # compile every csrc/*.hip, link libfp4x.so, then csrc/fp4x_host.cpp

Each translation unit compiles in a process of its own; the objects and the
libraries land next to this file (csrc/_build/, libfp4x.so, _fp4x_host.so).

libfp4x.so needs hipcc alone and is linked first: without torch it is all that
is built, and a host side that does not compile (no g++, no Python.h) is an
error behind it.
"""
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "_build")
LIB = os.path.join(HERE, "libfp4x.so")
HOST = os.path.join(HERE, "_fp4x_host.so")
ARCH = os.environ.get("FP4X_ARCH", "gfx950")

FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-ffp-contract=off",                      # fma only where the source asks for it
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",  # no packed fp32 VALU ops
    "-Wno-unused-command-line-argument",
]


def _hipcc():
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    cand = os.path.join(rocm, "bin", "hipcc")
    return cand if os.path.exists(cand) else shutil.which("hipcc")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _run(cmd, what):
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"{what}: {e}") from e
    if r.returncode != 0:
        raise RuntimeError(f"{what}:\n{r.stderr[-6000:]}")


def _host_object():
    """Compiles csrc/fp4x_host.cpp against the installed torch's headers: the
    object and torch's library folder, or None without torch."""
    src, obj = os.path.join(CSRC, "fp4x_host.cpp"), os.path.join(OBJ, "fp4x_host.o")
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    torch = spec.submodule_search_locations[0]
    inc = os.path.join(torch, "include")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-c", src, "-o", obj,
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f"-I{inc}",
           f"-I{os.path.join(inc, 'torch', 'csrc', 'api', 'include')}", f"-I{sysconfig.get_paths()['include']}",
           f"-I{os.path.join(os.environ.get('ROCM_PATH', '/opt/rocm'), 'include')}"]
    _run(cmd, f"{cmd[0]} failed for {src}")
    return obj, os.path.join(torch, "lib")


def _link_host(obj, torch_lib):
    tmp = HOST + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-fPIC", "-o", tmp, obj, f"-L{torch_lib}", "-lc10", "-lc10_hip",
           "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", f"-L{HERE}", "-l:libfp4x.so", "-Wl,-rpath,$ORIGIN"]
    _run(cmd, "link failed")
    os.replace(tmp, HOST)


def build(verbose=False, jobs=None):
    hipcc = _hipcc()
    if hipcc is None:
        raise RuntimeError("hipcc not found (set ROCM_PATH)")
    os.makedirs(OBJ, exist_ok=True)
    srcs = sources()

    def compile_one(src):
        obj = os.path.join(OBJ, os.path.basename(src)[:-4] + ".o")
        cmd = [hipcc, *FLAGS, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr[-6000:]}")
        if verbose:
            print(f"[fp4x build] {os.path.basename(src)}", flush=True)
        return obj

    with ThreadPoolExecutor(max_workers=jobs or min(8, len(srcs) + 1)) as ex:
        host = ex.submit(_host_object)
        objs = list(ex.map(compile_one, srcs))
    tmp = LIB + ".tmp"
    cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-4000:]}")
    os.replace(tmp, LIB)
    done = False
    try:
        built = host.result()
        if built is not None:
            _link_host(*built)
            done = True
        else:
            print("[fp4x build] no torch: _fp4x_host.so is not built", file=sys.stderr, flush=True)
    finally:
        if not done and os.path.exists(HOST):     # one of another build never stays beside the new library
            os.remove(HOST)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True, jobs=int(sys.argv[1]) if len(sys.argv) > 1 else None))
