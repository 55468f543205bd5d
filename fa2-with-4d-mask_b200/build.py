"""Builds libfa4d.so (the sm_100a kernels behind include/fa4d.h) and _fa4d_host.so (the host
binding of the operators around the attention) in place.

The library is compiled with nvcc for ``sm_100a`` only, the binding with the host compiler
against the installed torch (where there is none, it is left out: C callers do not need it), and
both are written next to this file, so they travel with the
source tree.  Objects go to ``_build/`` beside them.
Run ``python build.py`` (add ``--ptxas-info`` to print register / spill counts).
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
REPO = HERE.parent
CSRC = HERE / "csrc"
INCLUDE = REPO / "include"
BUILD = HERE / "_build"
LIB = HERE / "libfa4d.so"
HOST_SOURCE = CSRC / "fa4d_torch.cpp"
HOST_LIB = HERE / "_fa4d_host.so"

SOURCES = ["fa4d_api.cu", "fa4d_fwd.cu", "fa4d_bwd.cu", "fa4d_bwd256.cu", "fa4d_mask.cu", "fa4d_dq.cu", "fa4d_dq256.cu",
           "fa4d_rotary.cu", "fa4d_norm.cu", "fa4d_append.cu", "fa4d_decode.cu", "fa4d_decode8.cu", "fa4d_prefix.cu", "fa4d_evict.cu", "fa4d_cache_api.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put the CUDA toolkit on PATH)")


def _deps() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "fa4d.h"]


def _stale(target: Path, inputs: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(p.stat().st_mtime > t for p in inputs)


# Kernels that rebalance registers with setmaxnreg assume this exact allocation per
# thread at launch; fewer would make a setmaxnreg.inc wait forever.
LAUNCH_REGS = {"bwd_kernel": 128, "bwd256_kernel": 168, "fwd_kernel": 168, "prefix_kernel": 168}


def _check_launch_regs(src: Path, log: str) -> None:
    entry = None
    for line in log.splitlines():
        m = re.search(r"Compiling entry function '(\S+)'", line)
        if m:
            entry = m.group(1)
            continue
        m = re.search(r"Used (\d+) registers", line)
        if m and entry:
            for name, regs in LAUNCH_REGS.items():
                if name in entry and int(m.group(1)) != regs:
                    raise RuntimeError(f"{src.name}: {entry} uses {m.group(1)} registers, expected {regs}")
            entry = None


def _compile(nvcc: str, src: Path, obj: Path, ptxas_info: bool) -> str:
    cmd = [nvcc, *ARCH, *CFLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o", str(obj), "-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    _check_launch_regs(src, res.stdout + res.stderr)
    return res.stdout + res.stderr


def _build_host(force: bool) -> None:
    """The binding links libfa4d.so beside it and torch's own libraries (loaded by ``import
    torch`` before it); it is built again when its sources, or torch or Python, are others."""
    if importlib.util.find_spec("torch") is None:
        print(f"torch is not installed: {HOST_LIB.name} is not built", file=sys.stderr)
        return
    stamp = BUILD / "host_built_for.txt"
    target = f"torch {importlib.metadata.version('torch')}, python {sys.version_info.major}.{sys.version_info.minor}"
    known = stamp.read_text() if stamp.exists() else ""
    if not force and known == target and not _stale(HOST_LIB, [HOST_SOURCE, INCLUDE / "fa4d.h"]):
        return
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    tmp = HOST_LIB.with_suffix(".so.tmp")
    # The system's g++ (nvcc's host compiler): its libstdc++ is the one torch has loaded.
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{p}" for p in (root / "include", root / "include/torch/csrc/api/include", cuda / "include", INCLUDE,
                                sysconfig.get_paths()["include"])),
           str(HOST_SOURCE), "-o", str(tmp), f"-L{HERE}", "-l:libfa4d.so", f"-L{root / 'lib'}", "-ltorch_python",
           "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"host binding failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, HOST_LIB)
    stamp.write_text(target)


def build(force: bool = False, ptxas_info: bool = False, jobs: int | None = None) -> Path:
    nvcc = _nvcc()
    BUILD.mkdir(exist_ok=True)
    deps = _deps()
    todo = []
    for name in SOURCES:
        src = CSRC / name
        obj = BUILD / (src.stem + ".o")
        if force or ptxas_info or _stale(obj, [src, *deps]):
            todo.append((src, obj))
    logs = []
    if todo:
        with cf.ThreadPoolExecutor(max_workers=jobs or min(len(todo), os.cpu_count() or 1)) as ex:
            futs = [ex.submit(_compile, nvcc, s, o, ptxas_info) for s, o in todo]
            for f in futs:
                logs.append(f.result())
    objs = [BUILD / (Path(n).stem + ".o") for n in SOURCES]
    if force or todo or _stale(LIB, objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc, *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    _build_host(force)
    if ptxas_info:
        for log in logs:
            sys.stdout.write(log)
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true")
    ap.add_argument("-j", "--jobs", type=int, default=None)
    args = ap.parse_args()
    lib = build(force=args.force, ptxas_info=args.ptxas_info, jobs=args.jobs)
    print(lib)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
