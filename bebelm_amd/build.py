"""Builds libbebelm_moe.so (gfx950) in-tree from bebelm_amd/csrc/*.hip.

The library is the product: a C-ABI shared object (include/bebelm_moe.h). Flags:
  -ffp-contract=off                         no FMA contraction: f32 epilogues keep the
                                            reference's rounding sequence
  -fhip-fp32-correctly-rounded-divide-sqrt  IEEE f32 divide / sqrt (sigmoid, renorm, rmsnorm)
  -target-feature -packed-fp32-ops          no packed-FP32 instructions on this hardware pool
  -amdgpu-mfma-vgpr-form                    MFMA results in VGPRs (the GEMM epilogues read them
                                            with VALU; no accumulator-register copies); not where
                                            a wave has more than 256 registers to itself, of which
                                            the sums take the accumulator half
"""
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbebelm_moe.so")
SOURCES = ["bb_kernels.hip", "bb_decode.hip", "bb_prefill.hip", "bb_proj.hip", "bb_row1.hip", "bb_ops.hip",
           "bb_prompt_f32.hip", "bb_prompt_f16.hip", "bb_prompt_bf16.hip", "bb_prompt_kv4.hip", "bb_paged_prompt.hip",
           "bb_paged.hip", "bb_api.hip", "bb_gguf.hip"]
NO_VGPR_FORM = {"bb_prompt_f32.hip", "bb_prompt_f16.hip", "bb_prompt_bf16.hip", "bb_prompt_kv4.hip"}
ARCH = os.environ.get("BB_OFFLOAD_ARCH", "gfx950")


def hipcc():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "hipcc"


def flags():
    return [
        f"--offload-arch={ARCH}",
        "-O3",
        "-std=c++17",
        "-fPIC",
        "-ffp-contract=off",
        "-fhip-fp32-correctly-rounded-divide-sqrt",
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-Wall",
        "-Wno-unused-function",
    ]


def compile_one(src, obj, verbose):
    form = [] if os.path.basename(src) in NO_VGPR_FORM else ["-mllvm", "-amdgpu-mfma-vgpr-form"]
    cmd = [hipcc()] + flags() + form + ["-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    return subprocess.run(cmd, capture_output=True, text=True)


def build(verbose=False):
    srcs = [os.path.join(CSRC, s) for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    tmp = LIB + ".tmp"
    work = tempfile.mkdtemp(prefix="bebelm_build_")
    try:
        objs = [os.path.join(work, os.path.basename(s) + ".o") for s in srcs]
        jobs = min(len(srcs), int(os.environ.get("MAX_JOBS", os.cpu_count() or 1)), 8)
        with ThreadPoolExecutor(jobs) as pool:
            done = list(pool.map(lambda p: compile_one(*p, verbose), zip(srcs, objs)))
        bad = [r for r in done if r.returncode != 0]
        if not bad:
            done = [subprocess.run([hipcc(), f"--offload-arch={ARCH}", "-fPIC", "-shared"] + objs + ["-o", tmp],
                                   capture_output=True, text=True)]
            bad = [r for r in done if r.returncode != 0]
        if bad:
            sys.stderr.write("".join(r.stdout + r.stderr for r in bad))
            raise RuntimeError("hipcc failed building libbebelm_moe.so")
    finally:
        shutil.rmtree(work, ignore_errors=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
