"""Build recipe for libspk.so (sm_100a), in-tree.

Each ``csrc/*.cu`` file is compiled to an object with nvcc in parallel, then
linked into ``spikingtransformer_b200/libspk.so``.  The CUDA runtime is linked
statically; the driver API entry point used for TMA descriptors is resolved at
run time (``cudaGetDriverEntryPoint``), so the library needs no ``-lcuda``.
``csrc/embedding_autograd.cpp`` becomes the Python module ``_autograd.so`` beside
it, against the running torch's headers and libraries and ``libspk.so``.

    python -m spikingtransformer_b200.build [--force] [-j N]
"""

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libspk.so")
NODES = os.path.join(CSRC, "embedding_autograd.cpp")
NODES_LIB = os.path.join(PKG, "_autograd.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr",
         "-I" + INCLUDE]


def nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _compile(src, extra):
    obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
    cmd = [nvcc()] + ARCH + FLAGS + extra + ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed for %s:\n%s\n%s" % (src, " ".join(cmd), r.stderr[-8000:]))
    return obj, r.stderr


def needs_build():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(f) > t for f in _sources() + _headers() + [__file__])


def nodes_need_build():
    if not os.path.exists(NODES_LIB):
        return True
    t = os.path.getmtime(NODES_LIB)
    return any(os.path.getmtime(f) > t for f in [NODES, os.path.join(INCLUDE, "spk.h"), __file__])


def build_nodes(force=False):
    """Compile the autograd nodes (after libspk.so, which they are linked to)."""
    if not force and not nodes_need_build():
        return NODES_LIB
    import torch
    at = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    tmp = NODES_LIB + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
           "-I" + INCLUDE, "-I" + os.path.join(at, "include"),
           "-I" + os.path.join(at, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(cuda, "include"), NODES, "-o", tmp,
           "-L" + os.path.join(at, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-L" + PKG, "-lspk",
           "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for %s:\n%s\n%s" % (NODES, " ".join(cmd), r.stderr[-8000:]))
    os.replace(tmp, NODES_LIB)
    return NODES_LIB


def build(force=False, jobs=None, verbose=False, ptxas_info=False):
    """Compile every CUDA source for sm_100a, link libspk.so, then the autograd nodes (no-op
    where they are fresh)."""
    if force or needs_build():
        build_library(jobs, verbose, ptxas_info)
    build_nodes(force)
    return LIB


def build_library(jobs=None, verbose=False, ptxas_info=False):
    os.makedirs(BUILD, exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas_info else []
    srcs = _sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        results = list(ex.map(lambda s: _compile(s, extra), srcs))
    objs = [o for o, _ in results]
    if verbose or ptxas_info:
        for (o, err), s in zip(results, srcs):
            if err.strip():
                sys.stderr.write("== %s\n%s\n" % (os.path.basename(s), err))
    tmp = LIB + ".tmp"
    cmd = [nvcc()] + ARCH + ["-shared", "-cudart", "static", "-o", tmp] + objs
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n%s\n%s" % (" ".join(cmd), r.stderr[-8000:]))
    os.replace(tmp, LIB)
    return LIB


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=None)
    ap.add_argument("--ptxas-info", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.j, verbose=True, ptxas_info=a.ptxas_info))


if __name__ == "__main__":
    main()
