"""Builds libnemo_relpos.so in place: every CUDA source for sm_100a with
nvcc (-gencode arch=compute_100a,code=sm_100a -lineinfo), the C ABI host
code, statically linked against the CUDA runtime; and _nrp_torch, the
CPython/libtorch binding of the 8-bit linears and the LayerNorm, over it.

    python mlx-nemo-rs_b200/build.py [--force]
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libnemo_relpos.so")
BINDING_SRC = os.path.join(HERE, "torch_binding.cpp")
BINDING = os.path.join(HERE, "_nrp_torch" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
BINDING_STAMP = os.path.join(BUILD, "_nrp_torch.stamp")  # what it was built against
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         "--expt-relaxed-constexpr"]
SOURCES = ["gemm_sm100.cu", "gemm_tf32.cu", "attn_sm100.cu", "attn_simt.cu", "attn_stream.cu", "kernels_misc.cu",
           "noalloc.cu", "block_kernels.cu", "subsampling_kernels.cu", "api.cpp", "halo.cpp",
           "block.cpp", "subsampling.cpp", "fp8_quant.cu", "gemm_fp8.cu", "gemm_fp8_small.cu", "gemm_fp8_wgrad.cu",
           "norm_kernels.cu", "fp8_api.cpp"]


def _nccl_include():
    """Directory of nccl.h for halo.cpp (types and the config initializer
    only: the library is loaded with dlopen at run time).  The header of the
    NCCL that torch ships comes first, as that is the copy a torch process
    has loaded."""
    for base in (sysconfig.get_paths()["purelib"], sysconfig.get_paths()["platlib"]):
        d = os.path.join(base, "nvidia", "nccl", "include")
        if os.path.exists(os.path.join(d, "nccl.h")):
            return d
    for d in ("/usr/include", "/usr/local/cuda/include"):
        if os.path.exists(os.path.join(d, "nccl.h")):
            return d
    raise RuntimeError("nccl.h not found (needed to build halo.cpp)")


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, force):
    path = os.path.join(CSRC, src)
    obj = os.path.join(BUILD, src + ".o")
    headers = [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith((".h", ".cuh"))]
    headers.append(os.path.join(os.path.dirname(HERE), "include", "nemo_relpos.h"))
    if not force and not _stale(obj, [path] + headers):
        return obj, ""
    cmd = [NVCC, *ARCH, *FLAGS, "-c", path, "-o", obj]
    if src.endswith(".cpp"):
        cmd = [NVCC, *FLAGS, "-x", "c++", "-c", path, "-o", obj]
        if src == "halo.cpp":
            cmd[1:1] = ["-I", _nccl_include()]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj, r.stderr


def _torch_version(torch):
    """torch/version.py's __version__, without importing torch."""
    try:
        with open(os.path.join(torch, "version.py")) as f:
            return next(line.split("'")[1] for line in f if line.startswith("__version__"))
    except (OSError, StopIteration, IndexError):
        return "unknown"


def _build_binding(force):
    """The binding against the running interpreter's torch (its headers make
    this the slowest file: about a minute).  The C library and the host-side
    Python serve without it: where torch or its CUDA part or g++ is missing it
    is left out, and what needs it says so when it is asked for."""
    import importlib.util
    hdr = os.path.join(os.path.dirname(HERE), "include", "nemo_relpos.h")
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:
        return "torch is not installed: no binding"
    torch = os.path.dirname(spec.origin)
    libs = os.path.join(torch, "lib")
    cxx = shutil.which("g++")
    if not os.path.exists(os.path.join(libs, "libtorch_cuda.so")):
        return f"{torch} has no CUDA part: no binding"
    if cxx is None:
        return "no g++: no binding"
    stamp = f"torch {_torch_version(torch)} at {torch}\npython {sys.version}\n"
    try:
        with open(BINDING_STAMP) as f:
            same = f.read() == stamp
    except OSError:
        same = False
    if not force and same and not _stale(BINDING, [BINDING_SRC, hdr]):
        return ""
    inc = [os.path.join(torch, "include"),
           os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], "/usr/local/cuda/include"]
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-DTORCH_EXTENSION_NAME=_nrp_torch",
           *[f"-isystem{d}" for d in inc], BINDING_SRC, "-o", BINDING, f"-L{libs}", f"-L{HERE}",
           "-l:libnemo_relpos.so", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda",
           "-lc10", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libs}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    old = os.path.join(HERE, "_nrp_torch.so")  # (a name that any interpreter would load)
    if old != BINDING and os.path.exists(old):
        os.remove(old)
    with open(BINDING_STAMP, "w") as f:
        f.write(stamp)
    return r.stderr


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        results = list(ex.map(lambda s: _compile(s, force), SOURCES))
    objs = [o for o, _ in results]
    if verbose:
        for _, log in results:
            if log.strip():
                print(log)
    if force or _stale(LIB, objs):
        cmd = [NVCC, *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs, "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    log = _build_binding(force)
    if verbose and log.strip():
        print(log)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
