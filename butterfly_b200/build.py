"""Build libbna_b200.so (sm_100a) in-tree with nvcc, and the CPython binding of the paged cache.

    python -m butterfly_b200.build          # or __graft_entry__.build()

Each .cu under csrc/ is compiled to an object in csrc/_build/ (rebuilt when it or a
header is newer), then linked into butterfly_b200/libbna_b200.so.  csrc/binding.cpp becomes
butterfly_b200/_native.so (g++, against the installed torch's headers and libraries).
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import subprocess
import sys
import sysconfig
from importlib import metadata

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libbna_b200.so")
BUILD = os.path.join(CSRC, "_build")
BINDING = os.path.join(CSRC, "binding.cpp")
NATIVE = os.path.join(HERE, "_native.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
         "-Xptxas", "-v"]


def _headers():
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), _headers()):
        return obj
    cmd = [NVCC, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    with open(obj + ".ptxas.txt", "w") as f:
        f.write(r.stderr)
    if verbose:
        sys.stderr.write(r.stderr)
    return obj


def _build_binding() -> str:
    # what it was built against, beside the objects: another torch or Python may lay its types out anew
    stamp, built_for = os.path.join(BUILD, "_native.for"), f"torch {metadata.version('torch')}, python {sys.version}"
    if os.path.exists(NATIVE) and os.path.getmtime(NATIVE) >= max(os.path.getmtime(BINDING), _headers()) and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == built_for:
                return NATIVE
    import torch
    root = os.path.dirname(torch.__file__)
    inc, libs = os.path.join(root, "include"), os.path.join(root, "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", BINDING, "-o", NATIVE,
           f"-I{inc}", f"-I{inc}/torch/csrc/api/include", f"-I{sysconfig.get_path('include')}", f"-L{libs}",
           f"-Wl,-rpath,{libs}", "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {BINDING}:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(built_for)
    return NATIVE


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        native = ex.submit(_build_binding)
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
        native.result()
    if not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(o) for o in objs):
        cmd = [NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", OUT, *objs,
               "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
