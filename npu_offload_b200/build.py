"""Build libmoe_dp.so (the C-ABI library) in-tree with nvcc for sm_100a, and the torch side of the e4m3 and
balance-loss calls (_torch_binding.<Python>-torch<version>.so) with the host compiler.

    python -m npu_offload_b200.build [--force]

Both land next to this file, so they travel with the source tree to a GPU host; nothing is installed
into site-packages or a JIT cache.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libmoe_dp.so")
BINDING_SOURCE = os.path.join(CSRC, "torch_binding.cpp")
CXX = os.environ.get("CXX", "g++")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
SOURCES = ["moe_dp.cu", "route.cu", "experts.cu", "decode.cu", "noalloc.cu", "prefill.cu", "prefill_tc.cu",
           "block.cu", "fp8_quant.cu", "fp8_gemm.cu", "balance.cu"]


def cute_include():
    """CuTe / CUTLASS headers (descriptor and type definitions for the tcgen05 kernels): the header
    tree vendored with flashinfer, or $CUTLASS_INCLUDE."""
    cand = [os.environ.get("CUTLASS_INCLUDE", "")]
    try:
        import importlib.util
        spec = importlib.util.find_spec("flashinfer")
        if spec and spec.submodule_search_locations:
            cand.append(os.path.join(list(spec.submodule_search_locations)[0], "data", "cutlass", "include"))
    except Exception:
        pass
    for d in cand:
        if d and os.path.exists(os.path.join(d, "cute", "arch", "mma_sm100_desc.hpp")):
            return [d]
    raise RuntimeError("CuTe headers not found: set CUTLASS_INCLUDE to a CUTLASS include directory")


def sources():
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    deps = srcs + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    deps.append(os.path.join(ROOT, "include", "moe_dp.h"))
    return srcs, deps


def up_to_date():
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(d) <= t for d in sources()[1])


def binding_path():
    """Where the binding for the running Python and torch is: one of another version of either may differ in the
    layout of every object that it is handed, and is never loaded."""
    import torch
    return os.path.join(HERE, f"_torch_binding.{sys.implementation.cache_tag}-torch{torch.__version__}.so")


def build_binding(force=False):
    """Compiles the binding, linked to the library beside it, where it is older than what it is made of."""
    path = binding_path()
    deps = [BINDING_SOURCE, os.path.join(ROOT, "include", "moe_dp.h")]
    if not force and os.path.exists(path) and all(os.path.getmtime(d) <= os.path.getmtime(path) for d in deps):
        return path
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ext
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=_torch_binding"]
    for d in [*ext.include_paths(), sysconfig.get_paths()["include"]]:
        cmd += ["-isystem", d]
    cmd += [BINDING_SOURCE, "-o", path + ".tmp", *["-L" + d for d in ext.library_paths()], "-lc10", "-ltorch", "-ltorch_cpu",
            "-ltorch_python", "-L" + HERE, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    subprocess.check_call(cmd)
    os.replace(path + ".tmp", path)
    return path


def build(force=False, verbose=False, extra=(), out=None):
    """Builds the library (build_library) and, in-tree, the torch binding beside it.  The library needs neither torch nor
    a host compiler of its own: where the binding cannot be built, that is said on stderr."""
    lib = build_library(force, verbose, extra, out)
    if out is None:
        try:
            build_binding(force)
        except (ImportError, OSError, subprocess.CalledProcessError) as e:
            print(f"torch binding not built, the e4m3 and balance-loss calls need it: {e}", file=sys.stderr)
    return lib


def build_library(force=False, verbose=False, extra=(), out=None):
    """Compiles every source to an object in parallel (objects under _build/), then links the library.
    extra: additional nvcc flags; out: library path (default: the in-tree libmoe_dp.so)."""
    lib = out or LIB
    if not force and out is None and up_to_date():
        return lib
    srcs, _ = sources()
    tag = str(abs(hash((tuple(extra), lib))) % (1 << 32))
    objdir = os.path.join(HERE, "_build", tag)
    os.makedirs(objdir, exist_ok=True)
    common = [NVCC, *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
              "-I", os.path.join(ROOT, "include"), "-I", CSRC, *[a for d in cute_include() for a in ("-I", d)], *extra]
    if verbose:
        common.insert(1, "-Xptxas=-v")
    jobs = []
    for src in srcs:
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        cmd = [*common, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        jobs.append((obj, subprocess.Popen(cmd)))
    failed = [obj for obj, p in jobs if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, "nvcc " + " ".join(failed))
    link = [NVCC, *ARCH, "-shared", "-o", lib + ".tmp", *[obj for obj, _ in jobs], "-lcudart"]
    subprocess.check_call(link)
    os.replace(lib + ".tmp", lib)
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
