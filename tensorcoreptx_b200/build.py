"""In-tree build of the native libraries (nvcc, sm_100a only).

    python -m tensorcoreptx_b200.build          # build what is out of date
    python -m tensorcoreptx_b200.build --force  # rebuild everything

Outputs, next to this file:
    libtcgemm.so                 the C ABI of include/tcgemm.h (all kernels)
    _tcg_torch.so                the torch binding of the calls that are bound by
                                 the host when small (csrc/tcg_torch.cpp, g++)
    libtcgemm_compat_f16.so      reference-compatible C++ `launch_kernel` +
    libtcgemm_compat_s8.so       `Solver*` per precision (include/tcgemm_compat.h),
    libtcgemm_compat_s4.so       one per precision as the reference links one
                                 kernel file per binary
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ARCH + ["-O3", "-std=c++17", "-lineinfo", "-shared", "-Xcompiler", "-fPIC",
                 "-I" + INCLUDE]

LIB = os.path.join(HERE, "libtcgemm.so")
TORCH = os.path.join(HERE, "_tcg_torch.so")
COMPAT = {p: os.path.join(HERE, f"libtcgemm_compat_{p}.so") for p in ("f16", "s8", "s4")}


def _sources(*names):
    return [os.path.join(CSRC, n) for n in names]


def _deps():
    return [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".o")] + \
        [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def _includes(path, seen=None):
    """The files of this tree that `path` includes, itself among them."""
    seen = set() if seen is None else seen
    if path not in seen and os.path.exists(path):
        seen.add(path)
        for line in open(path):
            if line.startswith('#include "'):
                _includes(os.path.normpath(os.path.join(os.path.dirname(path), line.split('"')[1])), seen)
    return seen


def _compile(names, force, verbose):
    """Each source to an object file, those out of date side by side."""
    objects, running = [], []
    for src in _sources(*names):
        obj = src[:-3] + ".o"
        objects.append(obj)
        if force or _stale(obj, sorted(_includes(src))):
            cmd = [NVCC] + [f for f in COMMON if f != "-shared"] + ["-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            running.append((cmd, subprocess.Popen(cmd)))
    for cmd, p in running:
        if p.wait() != 0:
            raise subprocess.CalledProcessError(p.returncode, cmd)
    return objects


def _torch_command(out):
    import torch
    root = os.path.dirname(torch.__file__)
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"), sysconfig.get_paths()["include"], INCLUDE]
    return (["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + ["-I" + i for i in include] +
            _sources("tcg_torch.cpp") + ["-o", out, "-L" + os.path.join(root, "lib"), "-ltorch", "-ltorch_cpu",
                                         "-ltorch_python", "-lc10", "-lc10_cuda", "-L" + HERE, "-ltcgemm",
                                         "-Wl,-rpath,$ORIGIN"])


def build(force: bool = False, verbose: bool = True) -> list[str]:
    deps = _deps()
    built = []
    if force or _stale(LIB, deps):
        objects = _compile(("tcgemm.cu", "tcg_rows.cu"), force, verbose)
        _run([NVCC] + COMMON + objects + ["-o", LIB], verbose)
        built.append(LIB)
    defines = {"f16": "TCG_COMPAT_F16", "s8": "TCG_COMPAT_S8", "s4": "TCG_COMPAT_S4"}
    for prec, out in COMPAT.items():
        if force or _stale(out, deps + [LIB]):
            _run([NVCC] + COMMON + ["-D" + defines[prec]] + _sources("compat.cu") +
                 ["-L" + HERE, "-ltcgemm", "-Xlinker", "-rpath=$ORIGIN", "-o", out], verbose)
            built.append(out)
    if force or _stale(TORCH, [LIB] + sorted(_includes(*_sources("tcg_torch.cpp")))):
        _run(_torch_command(TORCH), verbose)
        built.append(TORCH)
    return built


if __name__ == "__main__":
    build(force="--force" in sys.argv)
