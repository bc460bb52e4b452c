"""In-tree build of the sm_100a CUDA library ``libpovs_sm100.so``.

Replaces the reference's setup.py template-instantiation build (setup.py:14-28,110-197):
the kernels here are runtime-general in (V, P, row bytes), so one library serves every
configuration and ``build_params.json`` records only the target architecture.
"""

from __future__ import annotations

import json
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC_DIR = PKG_DIR.parent / "csrc"
INCLUDE_DIR = PKG_DIR.parent.parent / "include"
LIB_NAME = "libpovs_sm100.so"
LIB_PATH = PKG_DIR / LIB_NAME
BUILD_PARAMS_PATH = PKG_DIR / "build_params.json"
CUDA_ARCH = "100a"

_HOST = [CSRC_DIR / "povs_host.h", INCLUDE_DIR / "povs.h"]
# Each source is compiled on its own (the shuffle kernels take minutes, the others seconds), with
# the headers whose change makes its object stale.
SOURCES = {
    CSRC_DIR / "povs_abi.cu": [*_HOST, CSRC_DIR / "povs_kernel.cuh", CSRC_DIR / "povs_rng.cuh",
                               CSRC_DIR / "povs_metrics.cuh", CSRC_DIR / "povs_mt19937.h"],
    CSRC_DIR / "povs_rows_abi.cu": [*_HOST, CSRC_DIR / "povs_rows.cuh", CSRC_DIR / "povs_sample.cuh"],
}
OBJECT_DIR = PKG_DIR.parent / "build"


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(cuda_home) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found: set CUDA_HOME or put nvcc on PATH")
    return found


def _flags(debug: bool) -> list[str]:
    flags = ["-gencode", f"arch=compute_{CUDA_ARCH},code=sm_{CUDA_ARCH}", "-lineinfo", "-std=c++17",
             "-Xcompiler", "-fPIC", "-O3"]
    return flags + (["-DPOVS_DEBUG=1"] if debug else [])


def _object(source: Path, debug: bool) -> Path:
    return OBJECT_DIR / f"{source.stem}{'_debug' if debug else ''}.o"


def _newer(target: Path, deps) -> bool:
    return target.exists() and all(d.stat().st_mtime <= target.stat().st_mtime for d in deps)


def is_stale() -> bool:
    deps = [d for source, headers in SOURCES.items() for d in (source, *headers)]
    return not BUILD_PARAMS_PATH.exists() or not _newer(LIB_PATH, deps)


def write_build_params(debug: bool = False) -> None:
    params = {
        "debug_mode": debug,
        "cuda_arch": [CUDA_ARCH],
        "vblock_sizes": [],
        "pblock_sizes": [],
        "instance_sizes": [],
        "cartesian_instancing": False,
        "instantiations": [],
        "instantiations_all_types": [],
    }
    BUILD_PARAMS_PATH.write_text(json.dumps(params, indent=2) + "\n")


def _run(cmd: list[str], output: Path, verbose: bool) -> None:
    """Run ``cmd + ["-o", <temporary>]`` and move the result to ``output``."""
    tmp = output.with_suffix(f"{output.suffix}.{os.getpid()}.tmp")
    cmd = [*cmd, "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, output)


def build(force: bool = False, verbose: bool = False, debug: bool = False) -> Path:
    """Compile the library in place (next to this file) unless it is up to date."""
    if force or is_stale():
        OBJECT_DIR.mkdir(exist_ok=True)
        stale = [s for s, headers in SOURCES.items() if force or not _newer(_object(s, debug), [s, *headers])]
        with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
            jobs = [pool.submit(_run, [_nvcc(), *_flags(debug), "-c", str(s)], _object(s, debug), verbose)
                    for s in stale]
            for job in jobs:
                job.result()
        _run([_nvcc(), *_flags(debug), "-shared", *(str(_object(s, debug)) for s in SOURCES)], LIB_PATH, verbose)
        write_build_params(debug)
    return LIB_PATH


if __name__ == "__main__":
    import sys

    build(force="--force" in sys.argv, verbose=True, debug="--debug" in sys.argv)
    print(LIB_PATH)
