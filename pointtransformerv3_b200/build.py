"""In-tree build of the CUDA library (nvcc, sm_100a only)."""
import glob
import os
import subprocess
import sys

from . import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(CSRC, "libptv3_b200.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "--use_fast_math", "-Xcompiler", "-fPIC"]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale(obj, src, deps):
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in [src] + deps)


def nodes_command():
    """The compiler call for the autograd nodes: a Python module against the headers and libraries of the torch that is installed, and the library."""
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    root = os.path.dirname(torch.__file__)
    include = cpp_extension.include_paths() + [sysconfig.get_paths()["include"], os.path.join(os.path.dirname(NVCC), "..", "include")]
    return (["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI]
            + [f for i in include for f in ("-isystem", i)]
            + [os.path.join(CSRC, "nodes.cpp"), "-o", _lib.nodes_path(), "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
               "-ltorch_python", "-L", CSRC, "-l:libptv3_b200.so", "-Wl,-rpath,$ORIGIN"])


def build(force=False, verbose=False):
    """Compiles every csrc/*.cu to an object and links libptv3_b200.so, then the module of autograd nodes."""
    hdrs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(
        os.path.join(HERE, "..", "include", "*.h"))
    objs, jobs = [], []
    for src in sources():
        obj = src[:-3] + ".o"
        objs.append(obj)
        if force or _stale(obj, src, hdrs):
            cmd = [NVCC] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
            jobs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = False
    for src, p in jobs:
        out = p.communicate()[0].decode()
        if p.returncode != 0 or verbose:
            sys.stderr.write("== %s\n%s\n" % (os.path.basename(src), out))
        failed |= p.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed")
    if jobs or not os.path.exists(LIB):
        subprocess.check_call([NVCC, "-shared", "-Wno-deprecated-gpu-targets", "-o", LIB] + objs + ["-lcudart"])
    if force or _stale(_lib.nodes_path(), os.path.join(CSRC, "nodes.cpp"), glob.glob(os.path.join(HERE, "..", "include", "*.h"))):
        subprocess.check_call(nodes_command())
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
