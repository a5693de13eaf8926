"""Builds the sm_100a shared library of the hot path (lib/libt8b.so) with nvcc.

bindings/operators.cpp becomes the Python module t8b/_operators.so, which links the installed torch and is
rebuilt when that changes. The library needs none of it: without torch it is built alone, and a module that
does not compile is reported once the library is linked.

Every .cu under csrc/ becomes one object; the engine translation unit is compiled with
--fmad=false (a fused multiply-add would round once where the reference CPU engine rounds
twice). Objects go to _build/ and are rebuilt when a source or header is newer.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from importlib import metadata
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
LIB = HERE / "lib" / "libt8b.so"
MODULE_SOURCE = HERE / "bindings" / "operators.cpp"
MODULE = HERE / "t8b" / "_operators.so"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
          f"-I{ROOT / 'include'}", f"-I{CSRC}"]
# Per-source extra flags.
EXTRA = {"sim.cu": ["--fmad=false"]}


def _newest_header() -> float:
    headers = list(CSRC.glob("*.cuh")) + list((ROOT / "include").glob("*.h"))
    return max((h.stat().st_mtime for h in headers), default=0.0)


def _module_command() -> list[str]:
    """The Python module of the torso operators, against the installed torch's headers and libraries."""
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    cuda = Path(NVCC).resolve().parent.parent
    includes = [*include_paths(), str(cuda / "include"), sysconfig.get_paths()["include"], str(ROOT / "include")]
    libraries = [flag for path in library_paths() for flag in (f"-L{path}", f"-Wl,-rpath,{path}")]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f"-I{path}" for path in includes), str(MODULE_SOURCE), "-o", str(MODULE), *libraries,
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def _module_job(verbose: bool):
    """What builds the Python module (None where it is up to date, or where there is no torch to link)."""
    stamp = BUILD / "operators.txt"
    try:
        against = f"torch {metadata.version('torch')} python {sys.version}"
        newest = max(MODULE_SOURCE.stat().st_mtime, (ROOT / "include" / "t8b.h").stat().st_mtime)
        if MODULE.exists() and MODULE.stat().st_mtime >= newest and stamp.exists() and stamp.read_text() == against:
            return None
        command = _module_command()
    except ImportError as missing:
        print(f"t8b/_operators.so is not built: {missing}", file=sys.stderr)
        return None
    if verbose:
        print(" ".join(command), flush=True)

    def run():
        subprocess.run(command, check=True)
        stamp.write_text(against)

    return run


def build(verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    LIB.parent.mkdir(exist_ok=True)
    newest_header = _newest_header()
    objects, commands = [], []
    for source in sorted(CSRC.glob("*.cu")):
        obj = BUILD / (source.stem + ".o")
        objects.append(obj)
        if obj.exists() and obj.stat().st_mtime >= max(source.stat().st_mtime, newest_header):
            continue
        cmd = [NVCC, *ARCH, *COMMON, *EXTRA.get(source.name, []), "-c", str(source), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        commands.append(cmd)
    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        compiled = [pool.submit(subprocess.run, cmd, check=True) for cmd in commands]
        job = _module_job(verbose)
        module = pool.submit(job) if job else None
        for done in compiled:
            done.result()
        if not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objects):
            cmd = [NVCC, *ARCH, "-shared", "-o", str(LIB), *map(str, objects), "-lcudart", "-lcuda", "-ldl"]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
        if module:
            module.result()
    return LIB


if __name__ == "__main__":
    build(verbose="-v" in sys.argv)
