"""Build libbattgp.so and libbattgp_products.so (HIP, gfx950 only) in-tree with hipcc.  No fallback of any kind.

    python -m battgp_amd.build [--force] [--experimental]

``--experimental`` builds a SECOND library, libbattgp_exp.so, from the same sources with -DBGP_EXPERIMENTAL: the default
library plus the optional kernel families no MI355X has timed yet (slim / split / fused panel chain, table-256 and
matrix-pipe fill interiors; bgp_internal.h).  The product never loads it unless BGP_EXPERIMENTAL_LIB=1 is set
(battgp_amd/_lib.py): it exists for the A/B stage of tools/gpu_session.sh and the optional parity cases."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbattgp.so")
LIB_EXPERIMENTAL = os.path.join(HERE, "libbattgp_exp.so")
SOURCES = ["bgp_fill.hip", "bgp_linalg.hip", "bgp_capi.hip"]
HEADERS = [os.path.join(CSRC, "bgp_internal.h"), os.path.join(CSRC, "bgp_fill_tile.inc"), os.path.join(os.path.dirname(HERE), "include", "battgp.h")]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function"]


# libbattgp_products.so: the products of battgp_amd/products.py (include/battgp_products.h)
PRODUCTS = os.path.join(CSRC, "products")
LIB_PRODUCTS = os.path.join(HERE, "libbattgp_products.so")
PRODUCTS_SOURCES = ["grouped.hip", "int8.hip"]
PRODUCTS_HEADERS = [os.path.join(PRODUCTS, h) for h in ("tile.h", "entry.h", "plan.h")] + [os.path.join(os.path.dirname(HERE), "include", "battgp_products.h")]
# no packed fp32 arithmetic: some of its forms have given wrong results on gfx950
PRODUCTS_FLAGS = FLAGS + ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


# _products_torch.so: what battgp_amd/products.py calls when nothing about a call is out of the ordinary (host code only)
TORCH_CALLS = os.path.join(PRODUCTS, "torch_calls.cpp")
LIB_TORCH_CALLS = os.path.join(HERE, "_products_torch.so")


def _hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: libbattgp.so cannot be built")


def needs_build(experimental: bool = False) -> bool:
    lib = LIB_EXPERIMENTAL if experimental else LIB
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    deps = [os.path.join(CSRC, s) for s in SOURCES] + HEADERS + [os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def build_lib(force: bool = False, verbose: bool = True, experimental: bool = False) -> str:
    lib = LIB_EXPERIMENTAL if experimental else LIB
    if not force and not needs_build(experimental):
        return lib
    _compile(CSRC, SOURCES, FLAGS + (["-DBGP_EXPERIMENTAL"] if experimental else []), ".exp.o" if experimental else ".o", lib, verbose)
    return lib


def build_products(force: bool = False, verbose: bool = True) -> str:
    deps = [os.path.join(PRODUCTS, s) for s in PRODUCTS_SOURCES] + PRODUCTS_HEADERS + [os.path.abspath(__file__)]
    if force or not os.path.exists(LIB_PRODUCTS) or any(os.path.getmtime(d) > os.path.getmtime(LIB_PRODUCTS) for d in deps):
        _compile(PRODUCTS, PRODUCTS_SOURCES, PRODUCTS_FLAGS, ".o", LIB_PRODUCTS, verbose)
    deps = [TORCH_CALLS, PRODUCTS_HEADERS[-1], os.path.abspath(__file__)]
    if force or not os.path.exists(LIB_TORCH_CALLS) or any(os.path.getmtime(d) > os.path.getmtime(LIB_TORCH_CALLS) for d in deps):
        _build_torch_calls(verbose)
    return LIB_PRODUCTS


def _build_torch_calls(verbose):
    import sysconfig

    try:
        import torch
    except ImportError:  # the C entries do without; battgp_amd.products says what it misses
        print(f"torch can not be imported: {os.path.basename(LIB_TORCH_CALLS)} is left out", file=sys.stderr)
        return

    root = os.path.dirname(torch.__file__)
    rocm = os.path.dirname(os.path.dirname(_hipcc()))
    cmd = [
        shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{sysconfig.get_paths()['include']}",
        "-isystem", os.path.join(root, "include"), "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
        "-isystem", os.path.join(rocm, "include"), TORCH_CALLS, "-o", LIB_TORCH_CALLS, f"-L{os.path.join(root, 'lib')}", f"-L{HERE}",
        "-l:libbattgp_products.so", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN",
    ]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def _compile(folder, sources, flags, suffix, lib, verbose):
    hipcc = _hipcc()
    from concurrent.futures import ThreadPoolExecutor

    def compile_one(src):
        obj = os.path.join(folder, src.replace(".hip", suffix))
        cmd = [hipcc, *flags, "-c", os.path.join(folder, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        return obj

    with ThreadPoolExecutor(len(sources)) as pool:  # the translation units side by side
        objs = list(pool.map(compile_one, sources))
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", lib]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)


if __name__ == "__main__":
    build_lib(force="--force" in sys.argv, experimental="--experimental" in sys.argv)
    build_products(force="--force" in sys.argv)
