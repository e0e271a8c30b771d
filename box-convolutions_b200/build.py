"""Builds the CUDA library for sm_100a and its PyTorch binding, in-tree:

    box-convolutions_b200/box_convolution/libboxconv_b200.so
    box-convolutions_b200/box_convolution/_torch_binding.<ABI>.so

The library: plain nvcc, no torch headers; its surface is the C ABI in include/boxconv_b200.h.
nvcc cross-compiles without a GPU.  Every source becomes an object under build/ of its own, made again when it, a
header of the repository that it includes, or the command that compiles it has changed; linked again when an object or
their list has.  The binding (csrc/*.cpp): g++ with torch's headers, linked against the library beside it.
Usage: python box-convolutions_b200/build.py [--force] [-v]
"""
import argparse
import concurrent.futures
import glob
import hashlib
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "box_convolution", "libboxconv_b200.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
]
OBJECTS = os.path.join(HERE, "build")

BINDING = os.path.join(HERE, "box_convolution", "_torch_binding" + sysconfig.get_config_var("EXT_SUFFIX"))
CXX = os.environ.get("CXX", "g++")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def newer(out, inputs):
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(f) < t for f in inputs + [os.path.abspath(__file__)])


def run(cmd, out, verbose):
    if verbose:
        print(" ".join(cmd))
    subprocess.check_call(cmd)
    os.replace(out + ".tmp", out)


def key(*what):
    return hashlib.sha256("\0".join(what).encode()).hexdigest()[:16]


def compile_object(compiler, src, force, verbose, also=""):
    """One source's object, and whether it had to be made; what it includes is read from the compiler's list.  Its name holds
    the command and `also`, what else it depends on: versions of headers outside the repository."""
    obj = os.path.join(OBJECTS, "%s.%s.o" % (os.path.basename(src), key(also, *compiler)))
    deps = obj + ".d"
    inputs = [src]
    if os.path.exists(deps):
        listed = open(deps).read().replace("\\\n", " ").split(":", 1)[1].split()
        inputs += [f for f in listed if os.path.abspath(f).startswith(os.path.dirname(HERE) + os.sep)]
    if not force and os.path.exists(deps) and all(map(os.path.exists, inputs)) and newer(obj, inputs):
        return obj, False
    shown = ["-Xptxas", "-v"] if verbose and compiler[0] == NVCC else []
    run(compiler + shown + ["-MMD", "-MF", deps, "-MT", obj, "-c", "-o", obj + ".tmp", src], obj, verbose)
    return obj, True


def compile_all(compiler, srcs, force, verbose, also=""):
    os.makedirs(OBJECTS, exist_ok=True)
    also += subprocess.check_output([compiler[0], "--version"], text=True)
    with concurrent.futures.ThreadPoolExecutor(max(1, os.cpu_count() or 1)) as pool:
        made = list(pool.map(lambda s: compile_object(compiler, s, force, verbose, also), srcs))
    return [o for o, _ in made], any(new for _, new in made)


def link(linker, libraries, out, objs, verbose):
    """Whether `out` had to be linked: beside the objects' times, the command of its last link counts."""
    command = linker + ["-o", out + ".tmp"] + objs + libraries
    note = os.path.join(OBJECTS, os.path.basename(out) + ".link")
    last = open(note).read() if os.path.exists(note) else ""
    if last == key(*command) and newer(out, objs):
        return False
    run(command, out, verbose)
    with open(note, "w") as f:
        f.write(key(*command))
    return True


def build_library(force=False, verbose=False):
    # (the largest sources first: they take minutes)
    srcs = sorted(sources(), key=os.path.getsize, reverse=True)
    objs, _ = compile_all([NVCC] + FLAGS, srcs, force, verbose)
    link([NVCC] + FLAGS + ["-shared"], [], OUT, objs, verbose)
    return OUT


def build_binding(force=False, verbose=False):
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(NVCC))
    dirs = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
            sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    libs = os.path.join(root, "lib")
    objs, _ = compile_all([CXX, "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
                             "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI] + ["-isystem" + d for d in dirs],
                          sorted(glob.glob(os.path.join(CSRC, "*.cpp"))), force, verbose,
                          also="torch %s, python %s" % (torch.__version__, sys.version))
    link([CXX, "-shared"],
         ["-L" + os.path.dirname(OUT), "-lboxconv_b200", "-L" + libs, "-lc10", "-lc10_cuda",
          "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + libs],
         BINDING, objs, verbose)
    return BINDING


def build(force=False, verbose=False):
    out = build_library(force, verbose)
    build_binding(force, verbose)
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    sys.exit(0)
