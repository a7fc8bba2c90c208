"""Build libnsdecode.so (HIP, gfx950) and its torch side _nsd_torch.so in-tree, with hipcc and g++.

-ffp-contract=off is part of the numerical contract: the decoder's fp32
log-softmax and fp64 score arithmetic must round operation by operation so
that results are reproducible on the host.
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
SO = PKG / "libnsdecode.so"
TORCH_SO = PKG / "_nsd_torch.so"
SOURCES = ["nsd_step.hip", "nsd_aux.hip", "nsd_prior.hip", "nsd_attn.hip", "nsd_seqattn.hip"]
TORCH_SOURCE = CSRC / "nsd_torch.cpp"
API = ROOT / "include" / "nsdecode.h"
HEADERS = [CSRC / "nsd_device.h", CSRC / "nsd_elem.h", API]
FLAGS = ["-O3", "--offload-arch=gfx950", "-ffp-contract=off", "-fPIC", "-std=c++17",
         "-fno-gpu-rdc", "-Wall", "-Wno-unused-function",
         # no packed fp32 instructions: some of their forms have given wrong results on these GPUs now and then
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(exe).exists():
        raise RuntimeError("hipcc not found: libnsdecode.so cannot be built")
    return exe


def _older(so: Path, sources) -> bool:
    return not so.exists() or any(p.stat().st_mtime > so.stat().st_mtime for p in sources)


def stale() -> bool:
    """Whether a source, a header or the flags (this file) changed since libnsdecode.so was built."""
    return _older(SO, [CSRC / s for s in SOURCES] + HEADERS + [Path(__file__)])


def torch_side_stale() -> bool:
    """The same of _nsd_torch.so, which also belongs to the torch that it was built against."""
    torch_version = Path(importlib.util.find_spec("torch").origin).parent / "version.py"
    return _older(TORCH_SO, [TORCH_SOURCE, API, Path(__file__), torch_version])


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True, cwd=str(CSRC))


def _build_kernels(verbose: bool) -> None:
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(len(SOURCES)) as pool:
        objs = [os.path.join(tmp, s + ".o") for s in SOURCES]
        list(pool.map(lambda so: _run([hipcc(), *FLAGS, f"-I{ROOT / 'include'}", f"-I{CSRC}", "-c", str(CSRC / so[0]),
                                       "-o", so[1]], verbose), zip(SOURCES, objs)))
        _run([hipcc(), "--offload-arch=gfx950", "-fPIC", "-shared", *objs, "-o", str(SO)], verbose)


def _build_torch_side(verbose: bool) -> None:
    import torch
    import torch.utils.cpp_extension as ext
    lib = Path(torch.__file__).parent / "lib"
    inc = [*ext.include_paths(), "/opt/rocm/include", sysconfig.get_path("include")]
    _run(["g++", "-O2", "-fPIC", "-shared", "-std=c++17", "-Wall", "-D__HIP_PLATFORM_AMD__",
          "-DTORCH_EXTENSION_NAME=_nsd_torch", *(a for i in inc for a in ("-isystem", i)), f"-I{ROOT / 'include'}",
          str(TORCH_SOURCE), "-o", str(TORCH_SO), f"-L{lib}", "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu",
          "-ltorch_python"], verbose)


def build(force: bool = False, verbose: bool = False) -> Path:
    jobs = []
    if force or stale():
        jobs.append(_build_kernels)
    if force or torch_side_stale():
        jobs.append(_build_torch_side)
    with ThreadPoolExecutor(2) as pool:
        list(pool.map(lambda job: job(verbose), jobs))
    return SO


if __name__ == "__main__":
    build(force=True, verbose=True)
    print(SO, os.path.getsize(SO), "bytes")
