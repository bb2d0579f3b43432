"""Builds libmomoe_b200.so (sm_100a only) in-tree with nvcc, and _native.so, its binding for torch tensors, with g++.

    python momoe-impl_b200/build.py            # -> momoe-impl_b200/momoe/libmomoe_b200.so, momoe-impl_b200/momoe/_native.so

nvcc cross-compiles, so this runs on machines without a GPU.  The library links cudart statically and
resolves the one driver entry point it needs at run time, so it also loads without a driver.
"""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
SOURCES = ["common.cu", "routing.cu", "grouped_gemm.cu", "decode_gemm.cu", "ep.cu",
           "norm.cu", "balance.cu", "fp8_gemm.cu", "fp8_decode.cu", "fp8_experts.cu"]
LIB_PATH = os.path.join(HERE, "momoe", "libmomoe_b200.so")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--threads", "4",
]


BINDING = os.path.join(CSRC, "binding.cpp")
BINDING_PATH = os.path.join(HERE, "momoe", "_native.so")
HEADER = os.path.join(HERE, "..", "include", "momoe_b200.h")


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def build(out=LIB_PATH, extra_flags=(), force=False, verbose=False):
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    deps = srcs + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    deps.append(HEADER)
    if out == LIB_PATH:
        build_binding(force=force, verbose=verbose)
    if not force and not _stale(out, deps):
        return out
    _run([nvcc, "-shared", "-o"], NVCC_FLAGS + list(extra_flags) + srcs, out, verbose)
    return out


def _run(head, tail, out, verbose):
    tmp = out + ".tmp%d" % os.getpid()     # written beside the target, then renamed: readers never see a partial file
    cmd = head + [tmp] + tail
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        if os.path.exists(tmp):
            os.remove(tmp)
        raise RuntimeError("%s failed building %s" % (os.path.basename(head[0]), out))
    os.replace(tmp, out)
    if verbose:
        sys.stderr.write(res.stdout + res.stderr)


def _built_for():
    """What a compiled binding fits; part of the binary, and compared again when the package loads it."""
    import torch
    return "torch %s, Python %d.%d" % (torch.__version__, *sys.version_info[:2])


def binding_stale(out=BINDING_PATH):
    if _stale(out, [BINDING, HEADER]):
        return True
    with open(out, "rb") as f:
        return _built_for().encode() + b"\0" not in f.read()


def build_binding(out=BINDING_PATH, force=False, verbose=False):
    """The torch binding; it takes the entry points from the loaded library at run time, so neither links the other."""
    if not force and not binding_stale(out):
        return out
    import torch
    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))
    flags = ["-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_native",
             '-DMOMOE_BUILT_FOR="%s"' % _built_for(),
             "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI)]
    includes = ["-isystem" + p for p in (os.path.join(home, "include"), os.path.join(cuda, "include"),
                                         os.path.join(home, "include", "torch", "csrc", "api", "include"),
                                         sysconfig.get_paths()["include"])]
    libs = ["-L" + os.path.join(home, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
            "-ltorch_python"]
    # the compiler on PATH and the C++ runtime that torch has loaded: a toolchain that links its own copy statically (CXX
    # may name one) puts two runtimes into the process, and the first error message crashes it
    _run(["g++", "-shared", "-o"], flags + includes + [BINDING] + libs + ["-l:libstdc++.so.6"], out, verbose)
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True,
                extra_flags=["-Xptxas", "-v"] if "--ptxas" in sys.argv else []))
