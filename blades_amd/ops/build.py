"""In-tree native builds (no hipify, no torch JIT cache).

* ``libblades_host.so``  — g++,  ``csrc/host.cpp``  (CPU; clustering, partitioner)
* ``libblades_hip.so``   — hipcc ``--offload-arch=gfx950``, every ``csrc/*.hip``

* ``_autograd.so``       — g++, ``csrc/autograd.cpp`` (no device code): the autograd
  nodes of ``ops/layers.py``, the one file that includes PyTorch's headers; it calls
  ``libblades_hip.so`` through addresses

The two libraries expose a plain C ABI and are loaded with ctypes, so neither needs
the PyTorch headers: a full rebuild is seconds, and hipcc cross-compiles gfx950
code objects on a machine without a GPU.
"""
import os
import re
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
HOST_LIB = HERE / "libblades_host.so"
HIP_LIB = HERE / "libblades_hip.so"
AUTOGRAD_LIB = HERE / "_autograd.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# scalar fp32 instructions only: some forms of the packed ones (v_pk_fma_f32 and its like), which -O3 makes of ordinary
# float code by itself, have given wrong results now and then (the host pass warns that it does not know the feature)
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _stale(target: Path, sources) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(Path(s).stat().st_mtime > t for s in sources)


def build_host(force: bool = False, verbose: bool = False) -> Path:
    srcs = [CSRC / "host.cpp"]
    if force or _stale(HOST_LIB, srcs):
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-o", str(HOST_LIB)] + [str(s) for s in srcs]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return HOST_LIB


def _headers(src: Path) -> list:
    """The headers of ``csrc`` that a source includes, directly or through another."""
    found, todo = [], [src]
    while todo:
        for name in re.findall(r'^#include "([^"]+)"', todo.pop().read_text(), re.M):
            h = CSRC / name
            if h.exists() and h not in found:
                found.append(h)
                todo.append(h)
    return found


def hip_sources():
    return sorted(CSRC.glob("*.hip"))


def build_hip(force: bool = False, verbose: bool = False, jobs: int = 4) -> Path:
    srcs = hip_sources()
    objdir = HERE / "_build"
    objdir.mkdir(exist_ok=True)
    procs = []
    objs = []
    for s in srcs:
        o = objdir / (s.stem + ".o")
        objs.append(o)
        if force or _stale(o, [s] + _headers(s)):
            cmd = [HIPCC, f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-c", str(s), "-o", str(o),
                   "-I", str(CSRC), "-Wno-unused-result"] + NO_PACKED_FP32
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((s, subprocess.Popen(cmd)))
            if len(procs) >= jobs:
                s0, p0 = procs.pop(0)
                if p0.wait() != 0:
                    raise RuntimeError(f"hipcc failed on {s0}")
    for s0, p0 in procs:
        if p0.wait() != 0:
            raise RuntimeError(f"hipcc failed on {s0}")
    if force or _stale(HIP_LIB, objs):
        cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(HIP_LIB)] + [str(o) for o in objs]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return HIP_LIB


def build_autograd(force: bool = False, verbose: bool = False) -> Path:
    src = CSRC / "autograd.cpp"
    if force or _stale(AUTOGRAD_LIB, [src] + _headers(src)):
        import sysconfig

        import torch
        from torch.utils.cpp_extension import include_paths

        lib = Path(torch.__file__).parent / "lib"
        rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
        inc = include_paths() + [f"{rocm}/include", sysconfig.get_paths()["include"]]
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
               "-DTORCH_EXTENSION_NAME=_autograd", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
        cmd += [a for i in inc for a in ("-isystem", i)] + [str(src), "-o", str(AUTOGRAD_LIB), f"-L{lib}", "-ltorch",
                                                            "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return AUTOGRAD_LIB


def build_all(force: bool = False, verbose: bool = True):
    build_host(force, verbose)
    build_hip(force, verbose)
    build_autograd(force, verbose)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
    print("built", HOST_LIB, HIP_LIB)
