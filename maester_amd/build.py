"""Build recipe of the HIP library (``libmaester_attn.so``) for gfx950.

``python -m maester_amd.build`` compiles every source under ``csrc/`` with hipcc and links them
into one shared object next to this file.  hipcc cross-compiles without a GPU.  Tests, the bench
and the smoke run only *load* the built library; they never build it.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "csrc", "build")
LIB_PATH = os.path.join(HERE, "libmaester_attn.so")

SOURCES = ["api.hip", "probe.hip", "tile_map.hip", "packed_ids.hip", "rmsnorm.hip", "cross_entropy.hip", "token_logprobs.hip", "linear_logprobs.hip", "linear_grads.hip", "adamw.hip", "prologue.hip", "attn_f32.hip", "attn_fwd_bf16.hip", "attn_fwd_pair_bf16.hip",
           "attn_bwd_bf16.hip"]

# -packed-fp32-ops is switched off on purpose: fp32 arithmetic is issued as scalar-per-lane VALU
# instructions only.
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffast-math", "-fno-finite-math-only",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
]

# sources whose results are those of their formulas in IEEE single precision, operation by operation (but for what they say)
EXACT_SOURCES = {"adamw.hip"}
EXACT_FLAGS = ["-fno-fast-math", "-ffp-contract=off"]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("hipcc not found")


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ_DIR, os.path.splitext(src)[0] + ".o")
    cmd = [_hipcc(), *HIPCC_FLAGS, *(EXACT_FLAGS if src in EXACT_SOURCES else []), "-c", os.path.join(CSRC, src), "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    err = "\n".join(l for l in res.stderr.splitlines() if "packed-fp32-ops" not in l)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{err}")
    if err.strip() and verbose:
        print(err, file=sys.stderr)
    return obj


def build(verbose: bool = False, jobs: int = 7) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), SOURCES))
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB_PATH, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
