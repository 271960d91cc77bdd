"""Build the sm_100a shared library ``_lib/libtelescope_b200.so`` and the host
extension ``_lib/_full_attention.so`` in place.

    python -m telescope_cache_b200.build_lib [--force]

Each ``csrc/*.cu`` is compiled by nvcc for ``sm_100a`` (in parallel, only when
it or a header changed) and linked into one shared library with a static
CUDA runtime.  The host extension (``csrc/host``, C++ against torch's headers)
calls the library's C entries.  Both travel with the source tree; nothing is
installed.
"""

import argparse
import glob
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OUT_DIR = os.path.join(PKG, "_lib")
LIB = os.path.join(OUT_DIR, "libtelescope_b200.so")
OBJ_DIR = os.path.join(ROOT, "_build")
HOST_SRC = os.path.join(CSRC, "host", "full_attention.cpp")
HOST_LIB = os.path.join(OUT_DIR, "_full_attention.so")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
         "--expt-relaxed-constexpr", "-Xptxas", "-O3"]


def nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the telescope_cache_b200 CUDA library cannot be built")


def _headers():
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def build_host(force=False):
    """Compile the host extension when its source or the C header changed."""
    header = os.path.join(ROOT, "include", "telescope_cache.h")
    if not force and os.path.exists(HOST_LIB) and \
            os.path.getmtime(HOST_LIB) >= max(os.path.getmtime(HOST_SRC), os.path.getmtime(header)):
        return HOST_LIB
    import torch
    from torch.utils import cpp_extension

    cuda_home = os.path.dirname(os.path.dirname(nvcc()))
    incs = cpp_extension.include_paths() + [os.path.join(cuda_home, "include"), sysconfig.get_paths()["include"]]
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    # the system compiler: $CXX may link its own C++ runtime in, and exceptions
    # then do not reach Python through torch's
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else shutil.which("g++") or "g++"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-o", HOST_LIB, HOST_SRC,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{i}" for i in incs],
           f"-L{torch_lib}", "-ltorch_python", "-ltorch", "-ltorch_cuda", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           f"-L{OUT_DIR}", "-l:libtelescope_b200.so", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{torch_lib}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {HOST_SRC}:\n{r.stdout}\n{r.stderr}")
    return HOST_LIB


def build(force=False, verbose=False):
    os.makedirs(OUT_DIR, exist_ok=True)
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr_time = _headers()
    cc = nvcc()

    def compile_one(src):
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        if (not force and os.path.exists(obj)
                and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_time)):
            return obj, None
        cmd = [cc, *ARCH, *FLAGS, "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
        return obj, (r.stdout + r.stderr) if verbose else None

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        results = list(ex.map(compile_one, srcs))
    objs = [o for o, _ in results]
    if verbose:
        for _, log in results:
            if log:
                sys.stdout.write(log)
    newest = max(os.path.getmtime(o) for o in objs)
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        cmd = [cc, *ARCH, "-shared", "-o", LIB, *objs, "-cudart", "static", "-lrt"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    build_host(force)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
