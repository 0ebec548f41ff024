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


def _text(cmd) -> str:
    """A command without the place it runs in: what a build depends on besides its sources."""
    return " ".join(str(c) for c in cmd).replace(str(HERE), ".")


def _stamp(target: Path) -> Path:
    return HERE / "_build" / (target.name + ".cmd")


def _stale(target: Path, sources, cmd=None) -> bool:
    """Is the target missing, older than a source, or (where one is given) made by another command?"""
    if not target.exists():
        return True
    t = target.stat().st_mtime
    if any(Path(s).stat().st_mtime > t for s in sources):
        return True
    if cmd is None:
        return False
    stamp = _stamp(target)
    return not stamp.exists() or stamp.read_text() != _text(cmd)


def _made(target: Path, cmd) -> None:
    _stamp(target).parent.mkdir(exist_ok=True)
    _stamp(target).write_text(_text(cmd))


def host_lib() -> Path:
    """What is built, for loading: made here only where it is missing or older than its source (an installed package has no
    record of the command)."""
    return build_host() if _stale(HOST_LIB, [CSRC / "host.cpp"]) else HOST_LIB


def build_host(force: bool = False, verbose: bool = False) -> Path:
    srcs = [CSRC / "host.cpp"]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-o", str(HOST_LIB)] + [str(s) for s in srcs]
    if force or _stale(HOST_LIB, srcs, cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        _made(HOST_LIB, cmd)
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


def build_hip(force: bool = False, verbose: bool = False, jobs: int = 8) -> Path:
    srcs = hip_sources()
    objdir = HERE / "_build"
    objdir.mkdir(exist_ok=True)
    procs = []
    objs = []

    def done(s0, o0, cmd0, p0):
        if p0.wait() != 0:
            raise RuntimeError(f"hipcc failed on {s0}")
        _made(o0, cmd0)

    for s in srcs:
        o = objdir / (s.stem + ".o")
        objs.append(o)
        cmd = [HIPCC, f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-c", str(s), "-o", str(o),
               "-I", str(CSRC), "-Wno-unused-result"] + NO_PACKED_FP32
        if force or _stale(o, [s] + _headers(s), cmd):
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((s, o, cmd, subprocess.Popen(cmd)))
            if len(procs) >= jobs:
                done(*procs.pop(0))
    for job in procs:
        done(*job)
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(HIP_LIB)] + [str(o) for o in objs]
    if force or _stale(HIP_LIB, objs, cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        _made(HIP_LIB, cmd)
    return HIP_LIB


def build_autograd(force: bool = False, verbose: bool = False) -> Path:
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths

    src = CSRC / "autograd.cpp"
    lib = Path(torch.__file__).parent / "lib"
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    inc = include_paths() + [f"{rocm}/include", sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-DTORCH_EXTENSION_NAME=_autograd", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cmd += [a for i in inc for a in ("-isystem", i)] + [str(src), "-o", str(AUTOGRAD_LIB), f"-L{lib}", "-ltorch",
                                                        "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"]
    made_of = cmd + ["#", torch.__version__]  # (the nodes are PyTorch's: another version's headers, another build)
    if force or _stale(AUTOGRAD_LIB, [src] + _headers(src), made_of):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        _made(AUTOGRAD_LIB, made_of)
    return AUTOGRAD_LIB


def build_all(force: bool = False, verbose: bool = True):
    build_host(force, verbose)
    build_hip(force, verbose)
    build_autograd(force, verbose)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
    print("built", HOST_LIB, HIP_LIB)
