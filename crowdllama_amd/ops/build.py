"""In-tree build of the HIP engine extension for gfx950.

Invoked by setup.py, __graft_entry__.build(), and lazily on first import
attempt. hipcc cross-compiles on CPU-only boxes; the resulting .so travels
with a copy of the tree to GPU machines (it is git-ignored).
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

OPS_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(OPS_DIR, "csrc")
ARCH = os.environ.get("CLA_GFX_ARCH", "gfx950")

# gfx950's packed float32 instructions (which -O3 forms by itself) have given
# wrong results now and then: no kernel is compiled with them
HIP_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# kvcache.hip's kernels work on every matrix product's result at once; results
# in accumulation registers cost a move each
FILE_FLAGS = {"kvcache.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]}

SOURCES = ["gguf.cpp", "engine.cpp", "testutil.cpp", "bindings.cpp",
           "kernels.hip", "mfma_probe.hip", "gemm.hip", "gemm_i8.hip",
           "kvcache.hip", "kv_bindings.cpp", "tokenizer.cpp"]


def _ext_suffix() -> str:
    return sysconfig.get_config_var("EXT_SUFFIX") or ".so"


def so_path() -> str:
    return os.path.join(OPS_DIR, "_core" + _ext_suffix())


def _newest_src_mtime() -> float:
    return max(os.path.getmtime(os.path.join(CSRC, s))
               for s in os.listdir(CSRC))


def needs_build() -> bool:
    so = so_path()
    return (not os.path.exists(so)) or os.path.getmtime(so) < _newest_src_mtime()


def build(verbose: bool = True, force: bool = False) -> str:
    so = so_path()
    if not force and not needs_build():
        return so
    import pybind11
    hipcc = os.environ.get("HIPCC", "hipcc")
    py_inc = sysconfig.get_paths()["include"]
    objs = []
    os.makedirs(os.path.join(OPS_DIR, "build"), exist_ok=True)
    procs = []
    for src in SOURCES:
        obj = os.path.join(OPS_DIR, "build", src.rsplit(".", 1)[0] + ".o")
        objs.append(obj)
        # (hipcc takes a .cpp for HIP too, and testutil.cpp has a kernel)
        cmd = [hipcc, *HIP_FLAGS, f"--offload-arch={ARCH}", "-O3",
               "-std=c++17", "-fPIC",
               *(["-DCLA_PERF_PROBE_NOATOMIC"] if os.environ.get("CLA_PROBE") else []),
               "-I", CSRC, "-I", py_inc, "-I", pybind11.get_include(),
               "-c", os.path.join(CSRC, src), "-o", obj]
        if src.endswith(".hip"):
            cmd[1:1] = ["-x", "hip", *FILE_FLAGS.get(src, [])]
        if verbose:
            print("[ops.build]", " ".join(cmd), file=sys.stderr)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                      stderr=subprocess.PIPE, text=True))
    for p, src in zip(procs, SOURCES):
        out, err = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"hipcc failed on {src}:\n{out}\n{err}")
        if verbose and err.strip():
            print(err, file=sys.stderr)
    link = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs,
            "-L/opt/rocm/lib", "-lrccl", "-o", so]
    if verbose:
        print("[ops.build]", " ".join(link), file=sys.stderr)
    r = subprocess.run(link, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc link failed:\n{r.stdout}\n{r.stderr}")
    return so


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(so_path())
