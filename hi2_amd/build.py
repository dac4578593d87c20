"""Build ``libhi2x.so`` (the gfx950 HIP library behind the C ABI in include/hi2x.h) and
``_tensors.so`` (host code: the addresses of many torch tensors in one call).

    python -m hi2_amd.build          # or hi2_amd.build.build()

Flags: -O3, no FP contraction (the reference rounds every product and sum
separately), IEEE-correct fp32 division and square root, no packed-fp32 code
generation, gfx950 only.
"""

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libhi2x.so")
SOURCES = ["api.hip", "gptq.hip", "ladder.hip", "format.hip", "hessian.hip", "chol.hip",
           "refine.hip", "stats.hip", "qad.hip", "packed.hip", "packed_few.hip",
           "packed_gemm.hip", "route.hip", "adamw.hip", "gated.hip", "grouped.hip",
           "grouped_tile.hip", "grouped_f32.hip",
           "grouped_few.hip"]
TENSORS = os.path.join(HERE, "_tensors.so")
ARCH = "gfx950"

OBJDIR = os.path.join(os.path.dirname(HERE), "_build")
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-fno-fast-math",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    return os.path.join(rocm, "bin", "hipcc")


def _run(cmd: list[str]) -> tuple[int, str]:
    r = subprocess.run(cmd, capture_output=True, text=True)
    out = "\n".join(
        line for line in (r.stdout + r.stderr).splitlines()
        if "packed-fp32-ops" not in line
    )
    return r.returncode, out


def tensors_command(out: str) -> list[str]:
    """The host compiler's command for ``csrc/tensors.cpp`` against torch's headers."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-I" + os.path.join(os.path.dirname(os.path.dirname(hipcc())), "include"),
           "-I" + sysconfig.get_paths()["include"], *("-I" + p for p in include_paths()),
           os.path.join(CSRC, "tensors.cpp"), "-o", out]
    for p in library_paths():
        cmd += ["-L" + p, "-Wl,-rpath," + p]
    return cmd + ["-ltorch_python", "-ltorch_cpu", "-lc10_hip", "-lc10"]


def build(verbose: bool = False, jobs: int | None = None) -> str:
    """Compile every HIP source into ``hi2_amd/libhi2x.so`` (always recompiles): one
    object per source, compiled in parallel under ``_build/``, then one link; and beside it
    ``hi2_amd/_tensors.so``."""
    os.makedirs(OBJDIR, exist_ok=True)
    objs = [os.path.join(OBJDIR, os.path.splitext(s)[0] + ".o") for s in SOURCES]
    cmds = [[hipcc(), *FLAGS, "-c", os.path.join(CSRC, s), "-o", o]
            for s, o in zip(SOURCES, objs)] + [tensors_command(TENSORS + ".tmp")]
    jobs = jobs or min(len(cmds), max(1, min(os.cpu_count() or 1, 16)))
    with ThreadPoolExecutor(jobs) as pool:
        results = list(pool.map(_run, cmds))
    for cmd, (rc, out) in zip(cmds, results):
        if verbose:
            print(" ".join(cmd), flush=True)
            if out.strip():
                print(out)
        if rc != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({rc}): {' '.join(cmd)}\n{out}")
    os.replace(TENSORS + ".tmp", TENSORS)
    tmp = LIB + ".tmp"
    rc, out = _run([hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp])
    if rc != 0:
        raise RuntimeError(f"link failed ({rc}):\n{out}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
