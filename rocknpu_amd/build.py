"""Build librocknpu_capi.so (the C ABI plus the gfx950 kernels) in-tree.

Every HIP source under csrc/ is compiled for gfx950 only with hipcc and linked
into rocknpu_amd/librocknpu_capi.so. Float semantics are pinned: no fast-math,
no FMA contraction, IEEE-correct f32 division, f32 denormals kept, and packed
FP32 instructions disabled.
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD_DIR = PKG / "_build"
LIB_NAME = "librocknpu_capi.so"
LIB_PATH = PKG / LIB_NAME

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

CFLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-fno-fast-math",
    "-fno-gpu-flush-denormals-to-zero",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # The leading scalar kernel arguments (up to 14 dwords) arrive preloaded in
    # SGPRs instead of through a scalar load from the argument segment at the
    # start of every wave: a graph-replayed launch's first loads go out
    # ~0.3 us earlier. Kernels list first the arguments their first loads
    # need; a struct passed by value is never preloaded.
    "-mllvm", "-amdgpu-kernarg-preload-count=14",
    "-Wall",
    "-Wno-unused-result",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]

SOURCES = ["repack.hip", "quant.hip", "gemm.hip", "gemm_skinny.hip", "gemv.hip", "gemv_mfma.hip", "gemv_tiled.hip", "launch.hip", "matmul.hip", "capi.hip", "sidecar.hip", "route.hip",
           "kv_cache.hip", "kv_stream.hip", "kv_prompt.hip", "kv_attention.hip"]


def _run(cmd: list[str]) -> None:
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    # hipcc's host pass does not know the packed-fp32-ops feature; that note is expected.
    noise = "'-packed-fp32-ops' is not a recognized feature"
    out = "\n".join(l for l in proc.stdout.splitlines() if noise not in l)
    if proc.returncode != 0:
        raise RuntimeError(f"command failed ({proc.returncode}): {' '.join(cmd)}\n{out}")
    if out.strip():
        sys.stderr.write(out + "\n")


def build(jobs: int = 6) -> Path:
    """Compile every source and link the shared library; returns its path."""
    BUILD_DIR.mkdir(exist_ok=True)
    objs = []
    cmds = []
    for src in SOURCES:
        obj = BUILD_DIR / (Path(src).stem + ".o")
        objs.append(obj)
        cmds.append([HIPCC, *CFLAGS, "-c", str(CSRC / src), "-o", str(obj)])
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        list(pool.map(_run, cmds))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)])
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build())
