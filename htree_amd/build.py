"""Builds libhtree_amd.so (gfx950) from htree_amd/csrc with hipcc, in-tree.

    python -m htree_amd.build          # compiles every time it is called
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(HERE, "libhtree_amd.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

SOURCES = ["htree_tree.hip", "htree_fwd.hip", "htree_fwd_stream.hip", "htree_fwd_wide_d32.hip",
           "htree_fwd_wide_d64.hip", "htree_fwd_wide_d128.hip", "htree_fwd_wide_d256.hip",
           "htree_bwd.hip", "htree_topk.hip", "htree_split.hip", "htree_cache.hip",
           "htree_draft_bf16.hip", "htree_draft_f16.hip", "htree_draft_f32.hip", "htree_verify.hip",
           "htree_pages.hip", "htree_norm.hip"]

# packed fp32 ops are disabled on purpose: some of their forms have given
# silently wrong results on these machines.
FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17", "-Wall",
    "-Wno-unused-function", "-Wno-unused-variable",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA accumulators in VGPRs: kernels that rotate an accumulator with
    # VALU between MFMAs otherwise copy it to and from AGPRs every tile
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    f"-I{INCLUDE}", f"-I{CSRC}",
]


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed ({' '.join(cmd)}):\n{r.stdout}\n{r.stderr}")
    return r


def build(verbose: bool = False) -> str:
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    objs = [os.path.join(objdir, os.path.splitext(s)[0] + ".o") for s in srcs]

    def compile_one(args):
        src, obj = args
        cmd = [HIPCC, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        _run(cmd)

    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        list(ex.map(compile_one, zip(srcs, objs)))
    tmp = LIB + ".tmp"
    _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp])
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
