"""Build recipe: ``libkdecay.so`` (one hipcc compilation per source for gfx950, then a link) and
``_native.so``, the host path of the Python functions (g++ against torch's headers).

Run ``python -m kilat_amd._build`` (or ``__graft_entry__.build()``).  The
library is written in-tree next to this file, where ``kilat_amd._lib`` loads it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SOURCES = [os.path.join(HERE, "csrc", name) for name in ("kdecay.hip", "kdecay_rows.hip", "gated_delta.hip", "attention.hip")]
INCLUDE = os.path.join(ROOT, "include")
LIBRARY = os.path.join(HERE, "libkdecay.so")
NATIVE_SOURCES = [os.path.join(HERE, "csrc", name) for name in ("native.cpp", "native_mixers.cpp")]
NATIVE = os.path.join(HERE, "_native.so")

# -packed-fp32-ops: no v_pk_*_f32 in the device code.
# -mcode-object-version=5: loadable by torch's bundled ROCm 7.0 runtime.
# No fast-math: fp32 division stays correctly rounded (hipcc's default), and
# the source turns fp contraction off itself.
HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-mcode-object-version=5",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(path):
        raise RuntimeError("hipcc not found (ROCm is required to build libkdecay.so)")
    return path


def _compile(jobs, what: str, verbose: bool) -> list:
    """Run the commands of (output, command) side by side; returns the outputs."""
    started = []
    for out, cmd in jobs:
        cmd = [*cmd, "-o", out]
        if verbose:
            print(" ".join(cmd), flush=True)
        started.append((out, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    done = [(out, proc.communicate()[0], proc.returncode) for out, proc in started]
    # hipcc's host pass does not know the packed-fp32 target feature and says
    # so; that line is expected and not shown.
    lines = [l for _, text, _ in done for l in text.splitlines() if "packed-fp32-ops" not in l and l.strip()]
    if any(rc != 0 for _, _, rc in done):
        raise RuntimeError(f"{what} failed:\n" + "\n".join(lines))
    if verbose and lines:
        print("\n".join(lines), flush=True)
    return [out for out, _, _ in done]


def build_library(verbose: bool = False) -> str:
    """Compile the csrc sources into libkdecay.so; returns the library path."""
    with tempfile.TemporaryDirectory(prefix="kdecay_build_") as work:
        objects = _compile([(os.path.join(work, os.path.basename(src) + ".o"),
                             [hipcc(), *HIPCC_FLAGS, "-I", INCLUDE, "-c", src]) for src in SOURCES], "hipcc", verbose)
        tmp = LIBRARY + ".tmp"
        _compile([(tmp, [hipcc(), "--offload-arch=gfx950", "-shared", *objects])], "hipcc", verbose)
        os.replace(tmp, LIBRARY)
    return LIBRARY


def build_native(verbose: bool = False) -> str:
    """Compile the host path into _native.so (after libkdecay.so, which it links); returns its path."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    base = ["g++", "-O2", "-std=c++17", "-fPIC", "-DUSE_ROCM", "-D__HIP_PLATFORM_AMD__=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE]
    for path in [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], "/opt/rocm/include"]:
        base += ["-isystem", path]
    with tempfile.TemporaryDirectory(prefix="kdecay_build_") as work:
        objects = _compile([(os.path.join(work, os.path.basename(src) + ".o"), [*base, "-c", src])
                            for src in NATIVE_SOURCES], "g++", verbose)
        cmd = ["g++", "-shared", *objects, "-L", HERE, "-lkdecay", "-Wl,-rpath,$ORIGIN"]
        for path in cpp_extension.library_paths():
            cmd += ["-L", path]
        cmd += ["-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"]
        tmp = NATIVE + ".tmp"
        _compile([(tmp, cmd)], "g++", verbose)
        os.replace(tmp, NATIVE)
    return NATIVE


def build(verbose: bool = False) -> None:
    build_library(verbose)
    build_native(verbose)


if __name__ == "__main__":
    build(verbose="-v" in sys.argv)
    print(LIBRARY, NATIVE)
