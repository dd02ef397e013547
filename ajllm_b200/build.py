"""Builds the sm_100a kernel library in-tree: ``python -m ajllm_b200.build``.

One ``nvcc -gencode arch=compute_100a,code=sm_100a`` invocation per ``.cu`` file (in parallel), then a
shared-library link into ``ajllm_b200/_native/libajllm_b200.so``. Objects are rebuilt only when their
source, a header or this file is newer, and the library is linked whenever an object is newer than it. ``-Xptxas -v``
output is kept next to the objects (``*.ptxas.txt``) so register and shared-memory use can be read without a GPU.
``csrc/fast_calls.cpp`` becomes a Python extension of its own, which knows torch's tensors and calls into the library. It
reads their C++ layout, so its file is named after the Python and torch it was built for and no other is loaded; the
framework works without it, and so a machine that cannot build it gets a warning.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE / "csrc"
OUT = PACKAGE / "_native"
LIB = OUT / "libajllm_b200.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xptxas", "-v", "--expt-relaxed-constexpr",
]
EXACT = {"logits"}          # compiled without fast math, which takes subnormal numbers for zero: their results are exact fp32 steps


def find_nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; the CUDA kernels cannot be built")
    return found


def fast_calls_path() -> Path:
    """Where the extension for this Python and this torch is."""
    import torch
    return OUT / f"fast_calls.{sys.implementation.cache_tag}.torch-{torch.__version__}.so"


def _needs_build(source: Path, obj: Path, headers: list[Path]) -> bool:
    if not obj.exists():
        return True
    stamp = obj.stat().st_mtime
    return any(dep.stat().st_mtime > stamp for dep in [source, *headers])


def _compile(nvcc: str, source: Path, obj: Path) -> tuple[Path, str]:
    cmd = [nvcc, *NVCC_FLAGS, *([] if source.stem in EXACT else ["--use_fast_math"]), "-I", str(CSRC), "-c", str(source), "-o", str(obj)]
    done = subprocess.run(cmd, capture_output=True, text=True)
    log = done.stdout + done.stderr
    obj.with_suffix(".ptxas.txt").write_text(log)
    if done.returncode != 0:
        raise RuntimeError(f"nvcc failed for {source.name}:\n{log[-6000:]}")
    return obj, log


def _into_place(command: list[str], target: Path) -> str | None:
    """Runs a compiler or linker whose output goes to ``target`` only if it succeeds; otherwise returns what it printed."""
    fresh = target.with_name(target.name + ".new")
    try:
        done = subprocess.run([*command, "-o", str(fresh)], capture_output=True, text=True)
    except OSError as error:
        return str(error)
    if done.returncode != 0:
        fresh.unlink(missing_ok=True)
        return (done.stdout + done.stderr)[-6000:]
    os.replace(fresh, target)
    return None


def _build_fast_calls() -> None:
    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = Path(find_nvcc()).resolve().parent.parent
    failure = _into_place(
        ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
         "-I", sysconfig.get_paths()["include"], "-I", str(root / "include"), "-I", str(root / "include/torch/csrc/api/include"),
         "-I", str(cuda / "include"), "-I", str(CSRC), str(CSRC / "fast_calls.cpp"),
         "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"], fast_calls_path())
    # one that is there was built from other sources, or for another Python or torch
    for old in OUT.glob("fast_calls*.so"):
        if failure is not None or old != fast_calls_path():
            old.unlink()
    if failure is not None:
        warnings.warn(f"g++ failed for fast_calls.cpp (small serving calls take longer without it):\n{failure}")


def build(force: bool = False, verbose: bool = False) -> Path:
    nvcc = find_nvcc()
    OUT.mkdir(parents=True, exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [Path(__file__).resolve()]          # (the flags are in here)
    jobs = []
    for source in sources:
        obj = OUT / (source.stem + ".o")
        if force or _needs_build(source, obj, headers):
            jobs.append((source, obj))
    if jobs:
        workers = min(len(jobs), max(1, (os.cpu_count() or 2)))
        with ThreadPoolExecutor(max_workers=workers) as pool:
            for obj, log in pool.map(lambda job: _compile(nvcc, *job), jobs):
                if verbose:
                    print(f"[build] {obj.name}\n{log}")
    objects = [OUT / (source.stem + ".o") for source in sources]
    if jobs or not LIB.exists() or LIB.stat().st_mtime < max(obj.stat().st_mtime for obj in objects):
        link = [nvcc, "-shared", *map(str, objects), "-gencode", "arch=compute_100a,code=sm_100a",
                "-lcudart_static", "-lpthread", "-ldl", "-lrt"]
        if (failure := _into_place(link, LIB)) is not None:
            raise RuntimeError(f"link failed:\n{failure}")
    if force or _needs_build(CSRC / "fast_calls.cpp", fast_calls_path(), [CSRC / "serving_args.h", Path(__file__).resolve()]):
        _build_fast_calls()
    return LIB


def main() -> None:
    force = "--force" in sys.argv
    path = build(force=force, verbose="-v" in sys.argv)
    print(path)


if __name__ == "__main__":
    main()
