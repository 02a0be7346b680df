"""Builds libyirage_hip.so (all HIP sources under csrc/) for gfx950 in-tree.

    python -m yirage_amd.build [--force]

Objects go to yirage_amd/_build/, the shared library next to this file, so
the built library travels with the source tree.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libyirage_hip.so")
ROOT = os.path.dirname(HERE)
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
HIPCC = os.path.join(ROCM, "bin", "hipcc")

FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Wno-unused-variable",
    "-Wno-unused-result",
    # no packed fp32 instructions anywhere in device code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I", os.path.join(ROOT, "include"),
]

# Per-source extra flags.  Attention keeps MFMA accumulators in VGPRs: its
# online-softmax rescale touches them between MFMAs, and AGPR-resident
# accumulators cost a copy in and out on every tile.
EXTRA = {
    "attention.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "graph_attn.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "sparse_attn.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "tree_attn.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    # the product kernel's small tiles copied AGPR accumulators in and out of every chunk
    "gemm_linear.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "gemm_norm.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "gemm_gated.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
}


def _deps_mtime() -> float:
    hdrs = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return max([os.path.getmtime(h) for h in hdrs] + [0.0])


def _compile(src: str, force: bool, hdr_t: float) -> str:
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    if not force and os.path.exists(obj):
        t = os.path.getmtime(obj)
        if t >= os.path.getmtime(src) and t >= hdr_t:
            return obj
    cmd = [HIPCC, *FLAGS, *EXTRA.get(os.path.basename(src), []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cc")))
    hdr_t = _deps_mtime()
    jobs = min(len(srcs), max(1, min(16, os.cpu_count() or 1)))
    with ThreadPoolExecutor(jobs) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, hdr_t), srcs))
    newest = max(os.path.getmtime(o) for o in objs)
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB, *objs, "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
