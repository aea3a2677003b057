"""Build the gfx950 shared library ``pratchya_amd/libpratchya_fp8.so`` and the
compiled binding of the row operators, ``pratchya_amd/_row_ops.so``.

The library is built in-tree with ``hipcc --offload-arch=gfx950`` so that it
travels with the source tree to the GPU machine; the binding holds no GPU code and
is built with the host compiler against torch's headers.  The library itself needs no
torch: where none is installed (another host of its C ABI), only the library is built.
Usage::

    python -m pratchya_amd.build          # or pratchya_amd.build.build()
"""
from __future__ import annotations

import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libpratchya_fp8.so"
ROW_OPS = PKG / "_row_ops.so"
SOURCES = ["quantize.hip", "quantize_t.hip", "gemm.hip", "gemm_t128.hip", "optim.hip", "elementwise.hip",
           "layer_norm.hip", "activation.hip", "logprobs.hip",
           "embedding.hip", "head_loss.hip", "linear_attention.hip"]

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CXX = os.environ.get("CXX", "g++")

# -packed-fp32-ops: keep the compiler from emitting v_pk_{add,mul,fma}_f32.
DEVICE_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def _run(cmd):
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in proc.stdout.splitlines()
                    if "packed-fp32-ops" not in l)  # host pass does not know the feature
    if proc.returncode != 0:
        raise RuntimeError(f"build failed ({proc.returncode}): {' '.join(cmd)}\n{out}")
    return out


def build(verbose: bool = False) -> Path:
    """Compile every HIP source for gfx950 and link the shared library."""
    build_dir = PKG / "_build"
    build_dir.mkdir(exist_ok=True)

    def compile_one(src: str) -> str:
        obj = build_dir / (Path(src).stem + ".o")
        out = _run([HIPCC, *DEVICE_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(CSRC / src), "-o", str(obj)])
        if verbose and out.strip():
            print(out)
        return str(obj)
    # side by side: one source after the other takes four times as long
    with ThreadPoolExecutor(min(8, len(os.sched_getaffinity(0)))) as pool:
        objs = list(pool.map(compile_one, SOURCES))
    tmp = LIB.with_suffix(".so.tmp")
    _run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", str(tmp)])
    os.replace(tmp, LIB)
    if importlib.util.find_spec("torch"):
        build_row_ops()
    else:
        ROW_OPS.unlink(missing_ok=True)      # of an older library
        print("no torch here: the Python binding of the row operators is not built", file=sys.stderr)
    return LIB


def build_row_ops() -> Path:
    """Compile the row operators' binding against this interpreter and its torch."""
    import torch
    torch_dir = Path(torch.__file__).resolve().parent
    include = torch_dir / "include"
    rocm = Path(HIPCC).resolve().parent.parent if "/" in HIPCC else Path("/opt/rocm")
    tmp = ROW_OPS.with_suffix(".so.tmp")
    _run([CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}", f"-I{include}",
          f"-I{include / 'torch' / 'csrc' / 'api' / 'include'}", f"-I{rocm / 'include'}",
          f"-I{sysconfig.get_paths()['include']}", str(CSRC / "row_ops.cpp"), "-o", str(tmp), f"-L{PKG}",
          f"-l:{LIB.name}", f"-L{torch_dir / 'lib'}", "-lc10", "-ltorch_cpu", "-ltorch_python", "-lc10_hip",
          "-ltorch_hip", "-Wl,-rpath,$ORIGIN"])
    os.replace(tmp, ROW_OPS)
    return ROW_OPS


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
