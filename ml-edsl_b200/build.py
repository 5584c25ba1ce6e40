"""Builds libb200edsl.so (all CUDA kernels + the C-ABI runtime) and
b200torch.so (the serving operators' calls on torch tensors) in-tree.

nvcc cross-compiles for sm_100a without a GPU, so this runs on any host with
the CUDA toolkit. Output: ml-edsl_b200/lib/.
"""
import os
import subprocess
import sys
import sysconfig
from importlib.metadata import PackageNotFoundError, version

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libb200edsl.so")
TORCH_SOURCE = os.path.join(CSRC, "torch_calls.cpp")
TORCH_LIB = os.path.join(LIBDIR, "b200torch.so")
TORCH_ABI = os.path.join(LIBDIR, "b200torch.abi")  # what it was compiled against
SOURCES = ["gemm_tf32x3.cu", "gemm_i32.cu", "gemm_i32_tc.cu", "elementwise.cu", "runtime.cu", "noalloc.cu", "reduce.cu", "peer.cu",
           "rms_norm.cu", "dense_w4.cu", "dense_w4_tc.cu", "token_logprobs.cu", "serving.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O3",
    "-shared",
    "--threads", "0",  # the sources side by side
]


def nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def torch_commands():
    """(compile, link) of the torch module; it finds libb200edsl.so beside it."""
    import torch
    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc())) or "/usr/local/cuda"
    obj = TORCH_LIB + ".o"
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    include = [os.path.join(base, "include"),
               os.path.join(base, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cxx = os.environ.get("CXX", "g++")
    compile_ = [cxx, "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={abi}"] + \
        ["-I" + d for d in include] + ["-c", TORCH_SOURCE, "-o", obj]
    link = [cxx, "-shared", obj, "-o", TORCH_LIB + ".tmp", "-L" + os.path.join(base, "lib"),
            "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda",
            "-L" + LIBDIR, "-lb200edsl", "-Wl,-rpath,$ORIGIN"]
    return compile_, link


def _stale(target):
    """Whether a source is newer than `target`, or there is none."""
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(HERE, "..", "include", "b200_edsl.h"))
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def torch_abi():
    """What the torch module is compiled against, without importing torch."""
    try:
        return f"torch {version('torch')}, {sys.implementation.cache_tag}"
    except PackageNotFoundError:
        return "no torch"


def _module_stale():
    """Also where the module is another torch's or Python's, or of unknown ones."""
    try:
        with open(TORCH_ABI) as f:
            built_for = f.read()
    except FileNotFoundError:
        built_for = None
    return _stale(TORCH_LIB) or built_for != torch_abi()


def needs_build():
    return _stale(LIB) or _module_stale()


def build(force=False, verbose=False, extra=()):
    """The library needs the CUDA toolkit alone: it is built first and stays where
    the torch module cannot be built (that is raised) or there is no torch (then
    mlir_edsl.serving is not to be had)."""
    lib, module = force or _stale(LIB), force or _module_stale()
    if not (lib or module):
        return LIB
    os.makedirs(LIBDIR, exist_ok=True)
    cmd = [nvcc()] + NVCC_FLAGS + list(extra) + [os.path.join(CSRC, s) for s in SOURCES] + [
        "-o", LIB + ".tmp", "-lpthread"]
    if verbose and lib:
        print(" ".join(cmd))
    compiling = subprocess.Popen(cmd) if lib else None
    failure, link = None, None
    try:  # beside nvcc
        if module:
            compile_, link = torch_commands()
            if verbose:
                print(" ".join(compile_), " ".join(link), sep="\n")
            subprocess.run(compile_, check=True)
    except ImportError:
        print("torch not found: mlir_edsl.serving is not built")
    except (OSError, subprocess.CalledProcessError) as e:
        failure = e
    finally:
        rc = compiling.wait() if compiling else 0
    if rc:
        raise subprocess.CalledProcessError(rc, cmd)
    if compiling:
        os.replace(LIB + ".tmp", LIB)
    if failure:
        raise failure
    if link:
        subprocess.run(link, check=True)
        os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
        os.remove(TORCH_LIB + ".o")
        with open(TORCH_ABI, "w") as f:
            f.write(torch_abi())
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True,
          extra=["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else [])
