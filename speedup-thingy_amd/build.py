"""Build librte_hip.so (gfx950) in-tree with hipcc, and librte_ops.so (autograd nodes over it) with the host compiler.

Usage: python speedup-thingy_amd/build.py [--jobs N]
The shared libraries land next to the Python package (rte_amd/librte_*.so) so
they travel with the source tree; no JIT cache, no site-packages install.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OUT = HERE / "rte_amd" / "librte_hip.so"
OPS = HERE / "rte_amd" / "librte_ops.so"
OBJ = HERE / "_build"
SOURCES = ["gemm.hip", "gemm_tile.hip", "route.hip", "norm.hip", "loss.hip", "shortlist.hip", "segreduce.hip", "glue.hip", "distill.hip", "macro.hip", "macro_fused.hip", "macro_cons.hip", "adamw.hip", "attention.hip", "noalloc.hip", "dispatch.hip", "svdsel.hip", "svd_fused.hip", "router.hip", "bookkeep.hip", "f32.hip", "replay.hip", "pool_fused.hip", "token_loss.hip", "head_loss.hip", "pool_balance.hip", "capi.hip"]

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # packed fp32 ops are kept out of the device code on purpose
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found; the ROCm toolchain is required to build librte_hip")


def _compile(src: Path, obj: Path) -> None:
    cmd = [_hipcc(), *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{proc.stderr[-6000:]}")


def _run(cmd: list[str], what: str) -> None:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{proc.stderr[-6000:]}")


def _torch_flags() -> tuple[list[str], list[str]]:
    """Compile and link flags for host code against the installed torch."""
    import torch

    root = Path(torch.__file__).resolve().parent
    abi = int(torch.compiled_with_cxx11_abi())
    include = [f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}"]
    return [f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *include], [f"-L{root / 'lib'}", "-ltorch", "-ltorch_cpu", "-lc10"]


def _compile_ops(obj: Path) -> None:
    cxx = os.environ.get("CXX") or "g++"
    _run([cxx, "-O2", "-std=c++17", "-fPIC", *_torch_flags()[0], "-c", str(CSRC / "loss_ops.cpp"), "-o", str(obj)],
         f"{cxx} for loss_ops.cpp")


def _link_ops(obj: Path) -> None:
    """librte_ops finds librte_hip beside itself; torch's libraries are those of the process."""
    tmp = OPS.with_suffix(".so.tmp")
    cxx = os.environ.get("CXX") or "g++"
    _run([cxx, "-shared", str(obj), f"-L{OUT.parent}", f"-l:{OUT.name}", *_torch_flags()[1], "-Wl,-rpath,$ORIGIN", "-o",
          str(tmp)], "link of librte_ops")
    os.replace(tmp, OPS)


def build(jobs: int | None = None, verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    objs = [OBJ / (Path(s).stem + ".o") for s in SOURCES]
    jobs = jobs or min(len(SOURCES), os.cpu_count() or 1)
    with cf.ThreadPoolExecutor(max_workers=jobs) as pool:
        futs = [pool.submit(_compile, CSRC / s, o) for s, o in zip(SOURCES, objs)]
        futs.append(pool.submit(_compile_ops, OBJ / "loss_ops.o"))
        for f in futs:
            f.result()
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr[-6000:]}")
    os.replace(tmp, OUT)
    _link_ops(OBJ / "loss_ops.o")
    if verbose:
        print(f"built {OUT} and {OPS.name}")
    return OUT


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args(argv)
    build(args.jobs, verbose=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
