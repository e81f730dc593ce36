"""Builds the HIP library ``libgqk.so`` in-tree for gfx950 (hipcc, no JIT cache).

    python hyperqwen-rtx4080s32_amd/gguf_hip/build.py     # as a script: no package import, so a
                                                          # stale or missing library is no obstacle
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)                      # hyperqwen-rtx4080s32_amd/
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
BUILD = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "libgqk.so")
# (source, extra flags, object): the GEMM is compiled once per token-block count, side by side
SOURCES = (("gqk_api.hip", (), "gqk_api.o"), ("gqk_codec.hip", (), "gqk_codec.o"), ("gqk_gemv.hip", (), "gqk_gemv.o"),
           ("gqk_mid.hip", (), "gqk_mid.o"), ("gqk_gemm_plan.hip", (), "gqk_gemm_plan.o"),
           *(("gqk_gemm.hip", (f"-DGQK_GEMM_MB={mb}",), f"gqk_gemm{mb}.o") for mb in (2, 4, 8)),
           ("gqk_gguf.cpp", (), "gqk_gguf.o"),
           *((f"gqk_{n}.hip", (), f"gqk_{n}.o") for n in ("lora", "rope", "attention", "pages")))
ARCH = os.environ.get("GQK_OFFLOAD_ARCH", "gfx950")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
MODULE = os.path.join(PKG, "_fast.so")   # the CPython module of the eager calls (gqk_torch.cpp)
FLAGS = [
    "-O3", "-fPIC", "-std=c++17", f"--offload-arch={ARCH}",
    "-I", os.path.join(REPO, "include"), "-I", CSRC,
    # packed fp32 VALU ops stay off (the pool's boxes have shown silent errors from them)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA accumulators in ordinary VGPRs (no v_accvgpr_read round trips in the GEMV epilogue)
    "-mllvm", "-amdgpu-mfma-vgpr-form",
]


def _run(cmd: list[str]) -> None:
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"hipcc failed ({p.returncode}): {' '.join(cmd)}\n{p.stderr[-6000:]}")


def _module_commands() -> tuple[list[str], list[str]]:
    """Compile and link of the eager calls' module against torch and the library beside it."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    obj = os.path.join(BUILD, "gqk_torch.o")
    compile_ = [HIPCC, "-x", "c++", "-O2", "-fPIC", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
                f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", os.path.join(REPO, "include"),
                *(x for d in [*include_paths(), "/opt/rocm/include", sysconfig.get_paths()["include"]] for x in ("-isystem", d)),
                "-c", os.path.join(CSRC, "gqk_torch.cpp"), "-o", obj]
    link = [HIPCC, "-shared", "-o", MODULE + ".tmp", obj, "-L", PKG, "-lgqk", "-Wl,-rpath,$ORIGIN",
            *(x for d in library_paths() for x in ("-L", d)), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python"]
    return compile_, link


def build(jobs: int | None = None) -> str:
    """Compile every source (HIP kernels; the host-only GGUF reader; the eager calls' module) and link libgqk.so and _fast.so (always
    rebuilds); returns the library path."""
    os.makedirs(BUILD, exist_ok=True)
    objs = []
    cmds = []
    for src, extra, name in SOURCES:
        obj = os.path.join(BUILD, name)
        objs.append(obj)
        cmds.append([HIPCC, *FLAGS, *extra, "-c", os.path.join(CSRC, src), "-o", obj])
    compile_module, link_module = _module_commands()
    cmds.append(compile_module)
    with ThreadPoolExecutor(max_workers=jobs or min(len(cmds), os.cpu_count() or 4)) as ex:
        list(ex.map(_run, cmds))
    tmp = LIB + ".tmp"
    _run([HIPCC, "-shared", f"--offload-arch={ARCH}", "-o", tmp, *objs])
    os.replace(tmp, LIB)
    _run(link_module)
    os.replace(MODULE + ".tmp", MODULE)
    return LIB


if __name__ == "__main__":
    print(build(int(sys.argv[1]) if len(sys.argv) > 1 else None))
