"""Builds ``libot_b200.so`` (the sm_100a kernels + the C ABI) in-tree with nvcc, and
``_tensors.so``, a small helper of the Python layer, with g++ against torch's headers.

Usage: ``python -m optimized_transducer_b200.build [-v]``.  The library links
the CUDA runtime statically and has no dependency on torch or Python.
"""
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libot_b200.so")
HELPER = os.path.join(HERE, "_tensors.so")
HELPER_STAMP = os.path.join(HERE, "_tensors.built")  # what HELPER was built for
HELPER_SOURCE = os.path.join(CSRC, "tensors.cc")
SOURCES = ["api.cu", "prep.cu", "logprob.cu", "lattice.cu", "gradient.cu", "noalloc.cu", "pack.cu",
           "exchange.cu", "fused_linear.cu", "fp8.cu", "sample.cu", "clip.cu"]
HEADERS = [os.path.join(CSRC, "ot_common.cuh"), os.path.join(CSRC, "tensor_core.cuh"),
           os.path.join(HERE, os.pardir, "include", "ot_b200.h")]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path():
    cand = shutil.which("nvcc") or os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    if not os.path.isfile(cand):
        raise RuntimeError("nvcc not found; it is needed to build libot_b200.so")
    return cand


def up_to_date():
    if not os.path.isfile(LIB):
        return False
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, s) for s in SOURCES] + HEADERS
    return all(os.path.getmtime(d) <= t for d in deps)


def built_for():
    """What the helper is tied to: it uses torch's and Python's C++ and C interfaces."""
    import torch

    return f"torch {torch.__version__}, Python {sys.version_info.major}.{sys.version_info.minor}"


def helper_up_to_date():
    if not (os.path.isfile(HELPER) and os.path.isfile(HELPER_STAMP)):
        return False
    t = os.path.getmtime(HELPER)
    if any(os.path.getmtime(d) > t for d in (HELPER_SOURCE, HEADERS[-1])):
        return False
    with open(HELPER_STAMP) as f:
        return f.read() == built_for()


def start_helper():
    """Starts the compilation of ``_tensors.so``."""
    import torch
    from torch.utils.cpp_extension import include_paths

    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DOT_BUILT_FOR="{built_for()}"', *[f"-I{p}" for p in (*include_paths(), sysconfig.get_paths()["include"], cuda)],
           HELPER_SOURCE, "-o", HELPER, f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def finish_helper(proc, verbose=False):
    out, _ = proc.communicate()
    if verbose or proc.returncode != 0:
        sys.stderr.write(out)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed on {HELPER_SOURCE}")
    with open(HELPER_STAMP, "w") as f:
        f.write(built_for())


def no_helper(why):
    warnings.warn(f"_tensors.so was not built ({type(why).__name__}: {why}); it needs g++, torch and the headers of both torch and Python. "
                  "The loss does without it; joiner_logits, sample_tokens, grad_norm and clip_grad_norm_ do not.", RuntimeWarning, stacklevel=3)


def build(force=False, verbose=False):
    """Compiles every kernel for sm_100a; returns the path of the library.  The library
    is what has to be there: where the helper cannot be built a warning says so, and
    what an earlier build left of it is gone."""
    helper = failed = None
    try:
        if force or not helper_up_to_date():
            for old in (HELPER, HELPER_STAMP):
                if os.path.isfile(old):
                    os.remove(old)
            helper = start_helper()
    except (ImportError, OSError, RuntimeError) as e:
        failed = e
    try:
        lib = build_library(force, verbose)
    finally:
        if helper is not None:
            try:
                finish_helper(helper, verbose)
            except RuntimeError as e:
                failed = e
    if failed is not None:
        no_helper(failed)
    return lib


def build_library(force=False, verbose=False):
    if not force and up_to_date():
        return LIB
    nvcc = nvcc_path()
    objs = []
    procs = []
    for src in SOURCES:
        obj = os.path.join(CSRC, src[:-3] + ".o")
        cmd = [nvcc, *ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
               "-ccbin", "g++", "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    for src, pr in procs:
        out, _ = pr.communicate()
        if verbose or pr.returncode != 0:
            sys.stderr.write(out)
        if pr.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}")
    link = [nvcc, *ARCH, "-shared", "-ccbin", "g++", "-o", LIB, *objs]
    subprocess.run(link, check=True)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose="-v" in sys.argv))
