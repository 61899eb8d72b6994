"""Build libnfx.so (the C-ABI library with every sm_100a kernel) in-tree.

    python -m neuroflow_b200.build [-v]

Compiles neuroflow_b200/csrc/*.cu and *.cpp with nvcc for sm_100a only
(-gencode arch=compute_100a,code=sm_100a), objects under _build/, and links
neuroflow_b200/libnfx.so, the nflow_infer command-line front-end and the torch front-end
_nfx_torch.so of neuroflow_b200.ops next to it.  The CUDA runtime is linked statically so the library does
not depend on which libcudart the host process (e.g. torch) loaded.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
from importlib import metadata

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(ROOT, "_build", "nfx")
LIB = os.path.join(PKG, "libnfx.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr",
         "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cpp")))


def _headers_mtime():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs.append(os.path.join(ROOT, "include", "nfx.h"))
    return max(os.path.getmtime(h) for h in hs if os.path.exists(h))


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    if (os.path.exists(obj) and os.path.getmtime(obj) >= os.path.getmtime(src)
            and os.path.getmtime(obj) >= _headers_mtime()):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
    if verbose and src.endswith(".cu"):
        cmd += ["-Xptxas", "-v"]
    if src.endswith(".cpp"):
        cmd += ["-x", "cu"] if False else []
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout or r.stderr):
        print(r.stdout + r.stderr, file=sys.stderr)
    return obj


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if (not os.path.exists(LIB)
            or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs)):
        cmd = [NVCC, *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs, "-lpthread", "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _build_cli()
    _build_torch()
    return LIB


TORCH_SRC = os.path.join(PKG, "torch_ext", "nfx_torch.cpp")
TORCH_EXT = os.path.join(PKG, "_nfx_torch.so")
TORCH_STAMP = os.path.join(OBJ, "_nfx_torch.made_for")  # the torch and Python that TORCH_EXT was built with


def _build_torch() -> None:
    """The compiled torch front-end of neuroflow_b200.ops (a Python module next to libnfx.so), with the
    headers and libraries of the installed torch; left out where torch is not installed (libnfx.so does not
    need it)."""
    try:
        made_for = f"torch {metadata.version('torch')} {sys.implementation.cache_tag}"
    except metadata.PackageNotFoundError:
        print("torch is not installed: without _nfx_torch.so (neuroflow_b200.ops)", file=sys.stderr)
        return
    hdr = os.path.join(ROOT, "include", "nfx.h")
    if (os.path.exists(TORCH_EXT) and os.path.getmtime(TORCH_EXT) >= max(os.path.getmtime(TORCH_SRC), os.path.getmtime(hdr))
            and os.path.exists(TORCH_STAMP) and open(TORCH_STAMP).read() == made_for):
        return
    import sysconfig

    import torch
    inc = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_nfx_torch",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + os.path.join(ROOT, "include"),
           "-isystem", inc, "-isystem", os.path.join(inc, "torch", "csrc", "api", "include"), "-isystem", cuda,
           "-isystem", sysconfig.get_paths()["include"], TORCH_SRC, "-o", TORCH_EXT, "-L" + PKG, "-lnfx",
           "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"torch front-end build failed:\n{r.stdout}\n{r.stderr}")
    with open(TORCH_STAMP, "w") as f:
        f.write(made_for)


CLI_SRC = os.path.join(PKG, "cli", "nflow_infer.cpp")
CLI = os.path.join(PKG, "nflow_infer")


def _build_cli() -> None:
    """The nflow_infer executable, linked against libnfx.so (found next to it)."""
    hpp = os.path.join(ROOT, "include", "nflow_runtime.hpp")
    if os.path.exists(CLI) and os.path.getmtime(CLI) >= max(os.path.getmtime(CLI_SRC),
                                                              os.path.getmtime(LIB),
                                                              os.path.getmtime(hpp)):
        return
    cmd = ["g++", "-std=c++17", "-O2", "-I" + os.path.join(ROOT, "include"), CLI_SRC, "-o", CLI,
           "-L" + PKG, "-lnfx", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nflow_infer build failed:\n{r.stdout}\n{r.stderr}")


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
