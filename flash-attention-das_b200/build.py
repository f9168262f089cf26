"""Build libfa_b200.so (sm_100a only) in-tree with nvcc, and beside it _fa_b200_host.so, the compiled host part of the
bounded-cache calls, against the installed torch.  Usage: python build.py [--force] [--verbose] [--test-hooks]

--test-hooks builds libfa_b200_testhooks.so beside it: the same sources with -DFA_B200_TEST_HOOKS (device-side waits
give up after about a millisecond, and one entry lets a launch withhold a tile load).  Only the failure-detection
tests load that library; the product never does."""
import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libfa_b200.so")
OUT_HOST = os.path.join(HERE, "_fa_b200_host.so")
HOST_KEY = os.path.join(HERE, "build", "_fa_b200_host.key")   # host_key() of the module that was built last
OUT_HOOKS = os.path.join(HERE, "libfa_b200_testhooks.so")
SOURCES = ["fa_api.cu", "fa_combine.cu", "fa_decode.cu", "fa_prefill.cu", "fa_prefill_pair.cu", "fa_prefill_dense.cu", "fa_kv_append.cu", "fa_glue.cu", "fa_block_select.cu", "fa_exchange.cu", "fa_page_select.cu", "fa_kv_evict.cu", "fa_token_weights.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "--use_fast_math",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]


def _deps(out):
    host = os.path.join(CSRC, "fa_host.cpp")
    files = [host] if out == OUT_HOST else [f for f in (os.path.join(CSRC, n) for n in os.listdir(CSRC)) if f != host]
    files.append(os.path.join(os.path.dirname(HERE), "include", "fa_b200.h"))
    return files


def host_key():
    """What the host module is built for, in full: a pre-release or vendor build of torch has a C++ ABI of its own."""
    import torch
    return "torch %s, Python %s" % (torch.__version__, sysconfig.get_config_var("SOABI"))


def _built_for():
    try:
        with open(HOST_KEY) as f:
            return f.read()
    except OSError:
        return None


def needs_build(out=OUT):
    if not os.path.exists(out):
        return True
    if out == OUT_HOST and _built_for() != host_key():
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(f) > t for f in _deps(out))


def build_host(force=False):
    """The Python module of csrc/fa_host.cpp: C++ only, no CUDA source."""
    if not force and not needs_build(OUT_HOST):
        return OUT_HOST
    import torch
    base = os.path.dirname(torch.__file__)
    part = OUT_HOST + ".%d" % os.getpid()
    key = host_key()
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
           '-DFA_B200_HOST_KEY="%s"' % key, "-I" + os.path.join(base, "include"), "-I" + os.path.join(base, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"),
           os.path.join(CSRC, "fa_host.cpp"), "-o", part, "-L" + os.path.join(base, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for fa_host.cpp:\n%s\n%s" % (r.stdout, r.stderr))
    os.replace(part, OUT_HOST)
    os.makedirs(os.path.dirname(HOST_KEY), exist_ok=True)
    with open(HOST_KEY, "w") as f:
        f.write(key)
    return OUT_HOST


def build(force=False, verbose=False, test_hooks=False):
    """The library, and the host module where there is a torch to build it against (the C ABI needs none)."""
    out = build_library(force, verbose, test_hooks)
    if not test_hooks:
        if importlib.util.find_spec("torch"):
            build_host(force)
        else:
            sys.stderr.write("no torch: %s is not built\n" % OUT_HOST)
    return out


def build_library(force=False, verbose=False, test_hooks=False):
    out = OUT_HOOKS if test_hooks else OUT
    if not force and not needs_build(out):
        return out
    objdir = os.path.join(HERE, "build", "testhooks" if test_hooks else "")
    os.makedirs(objdir, exist_ok=True)
    extra = ["-Xptxas", "-v"] if verbose else []
    if test_hooks:
        extra.append("-DFA_B200_TEST_HOOKS")

    def compile_one(src):
        obj = os.path.join(objdir, src.replace(".cu", ".o"))
        cmd = [NVCC, *FLAGS, *extra, "-c", os.path.join(CSRC, src), "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed for %s:\n%s\n%s" % (src, r.stdout, r.stderr))
        if verbose:
            sys.stderr.write(r.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=6) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    cmd = [NVCC, "-shared", "-o", out, *objs, "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n%s\n%s" % (r.stdout, r.stderr))
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, test_hooks="--test-hooks" in sys.argv))
