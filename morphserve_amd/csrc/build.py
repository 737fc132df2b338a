"""Build the C-ABI HIP libraries in-tree with hipcc for gfx950.

``libmorphkv.so`` is the product: it exports exactly what ``include/morphkv.h`` declares.
``libmorphkv_diag.so`` is its diagnostic twin, built from the same sources with ``-DMKV_DIAG=1``
plus ``diag.hip``: the same entry points and, on top, the switches and measurement hooks of
``include/morphkv_diag.h`` (kernel variants, per-launch event timing, per-workgroup time stamps,
calibration loops).  Benchmarks and tests that need those load the twin; the package never does.

``_binding`` (with the interpreter's tag in its file name) is the host side of the 8-bit cache's and the rotary
operators: argument checks and the call, a CPython module over torch's C++ tensors; it holds no kernel and takes the
library's entries by address.

Usage: ``python -m morphserve_amd.csrc.build`` or ``build_library()``.
The shared objects land next to the sources so that they travel with the tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "libmorphkv.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
DIAG_LIB_PATH = os.path.join(HERE, "libmorphkv_diag.so")
BINDING_PATH = os.path.join(HERE, "_binding" + sysconfig.get_config_var("EXT_SUFFIX"))

SOURCES = [
    "core.hip",
    "kv_append.hip",
    "rope.hip",
    "rotary.hip",
    "kv8_store.hip",
    "attn8_decode.hip",
    "attn8_prefill.hip",
    "paged_attn_decode.hip",
    "prefill_attn.hip",
    "block_pool.hip",
    "migrate.hip",
    "vmm_arena.hip",
]
DIAG_SOURCES = SOURCES + ["diag.hip"]

# -packed-fp32-ops is switched off: the compiler must not form v_pk_*_f32.
HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-fno-gpu-rdc",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I" + INCLUDE,
    "-I" + HERE,
]


def _hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found; the morphkv library cannot be built")
    return exe


def _compile(src: str, obj_dir: str, defines=()) -> str:
    obj = os.path.join(obj_dir, os.path.splitext(src)[0] + ".o")
    cmd = [_hipcc(), *HIPCC_FLAGS, *defines, "-c", os.path.join(HERE, src), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{res.stderr}")
    return obj


def _build_binding() -> None:
    from torch.utils.cpp_extension import include_paths
    import torch
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = BINDING_PATH + ".tmp"
    cmd = [_hipcc(), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-x", "c++",
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-I" + INCLUDE,
           "-I" + os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_hipcc()))), "include"),
           *("-I" + p for p in include_paths()), "-I" + sysconfig.get_paths()["include"],
           os.path.join(HERE, "binding.cpp"), "-o", tmp, "-L" + libs, "-ltorch_python", "-ltorch_cpu", "-ltorch_hip",
           "-lc10", "-lc10_hip"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for binding.cpp:\n{res.stderr}")
    os.replace(tmp, BINDING_PATH)


def _link(objs, out: str) -> None:
    tmp = out + ".tmp"
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC",
           "-Wl,--version-script=" + os.path.join(HERE, "exports.map"), "-o", tmp, *objs]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, out)


def build_library(verbose: bool = True, jobs: int = 8, diag: bool = True) -> str:
    """Compile every source and link ``libmorphkv.so`` (and, with ``diag``, its diagnostic twin)
    and the ``_binding`` module; always rebuilds."""
    obj_dir = os.path.join(HERE, "build")
    diag_dir = os.path.join(obj_dir, "diag")
    os.makedirs(diag_dir if diag else obj_dir, exist_ok=True)
    work = [(s, obj_dir, ("-DMKV_DIAG=0",)) for s in SOURCES]
    if diag:
        work += [(s, diag_dir, ("-DMKV_DIAG=1",)) for s in DIAG_SOURCES]
    # the attention files dominate the build: start them first
    work.sort(key=lambda w: 0 if "attn" in w[0] else 1)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        binding = ex.submit(_build_binding)
        objs = list(ex.map(lambda w: (w[1], _compile(*w)), work))
    _link([o for d, o in objs if d == obj_dir], LIB_PATH)
    if diag:
        _link([o for d, o in objs if d == diag_dir], DIAG_LIB_PATH)
    binding.result()                        # the libraries need neither Python nor torch: they are there if this fails
    if verbose:
        for path in (LIB_PATH, DIAG_LIB_PATH, BINDING_PATH) if diag else (LIB_PATH, BINDING_PATH):
            print(f"built {path} ({os.path.getsize(path) / 1024:.0f} KiB)")
    return LIB_PATH


if __name__ == "__main__":
    build_library()
    sys.exit(0)
