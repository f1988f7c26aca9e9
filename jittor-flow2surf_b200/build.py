"""Build libflow2surf_sm100.so from csrc/*.cu with nvcc for sm_100a.

Objects go to _build/ beside this file; the shared library lands inside the
Python package (flow2surf_b200/libflow2surf_sm100.so) so that it travels with
the source tree, and so does the PyTorch binding of the 8-bit feed-forward
operators (flow2surf_b200/_feedforward.so, from csrc/feedforward_torch.cpp with
the host compiler). Only sources newer than their object (or than any header)
are recompiled. The library needs nvcc alone; where torch, Python's headers or
g++ are missing, the binding is left out with a message.

    python jittor-flow2surf_b200/build.py [--force] [--jobs N]
"""

from __future__ import annotations

import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
INCLUDE = ROOT / "include"
BUILD = HERE / "_build"
LIBRARY = HERE / "flow2surf_b200" / "libflow2surf_sm100.so"
BINDING_SOURCE = CSRC / "feedforward_torch.cpp"
BINDING = HERE / "flow2surf_b200" / "_feedforward.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    *ARCH,
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler",
    "-fPIC",
    "-Xptxas",
    "-warn-spills",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(path).exists():
        raise RuntimeError("nvcc not found; the CUDA 12.9 toolkit is required")
    return path


def _newest_header() -> float:
    headers = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in headers), default=0.0)


def _compile(src: Path, force: bool, extra: list[str]) -> tuple[Path, str]:
    obj = BUILD / (src.stem + ".o")
    if not force and obj.exists():
        if obj.stat().st_mtime >= max(src.stat().st_mtime, _newest_header()):
            return obj, ""
    cmd = [nvcc(), *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{proc.stdout}\n{proc.stderr}")
    return obj, proc.stderr


def binding_lacks() -> str | None:
    """What the PyTorch binding cannot be built for, or None."""
    if importlib.util.find_spec("torch") is None:
        return "torch is not installed for this interpreter"
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return "Python.h is not installed"
    if shutil.which("g++") is None:
        return "g++ not found"
    return None


def _compile_binding(force: bool) -> tuple[Path, str]:
    """Object of the PyTorch binding, against the torch of this interpreter (a
    stamp beside it names their versions)."""
    import torch

    obj, stamp = BUILD / "feedforward_torch.o", BUILD / "feedforward_torch.stamp"
    wanted = f"{torch.__version__} {sys.version}"
    newest = max(i.stat().st_mtime for i in (BINDING_SOURCE, *INCLUDE.glob("*.h")))
    if (not force and obj.exists() and stamp.exists() and stamp.read_text() == wanted
            and obj.stat().st_mtime >= newest):
        return obj, ""
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{INCLUDE}", "-isystem", str(root / "include"),
           "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(cuda / "include"),
           "-c", str(BINDING_SOURCE), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDING_SOURCE.name}:\n{proc.stdout}\n{proc.stderr}")
    stamp.write_text(wanted)
    return obj, proc.stderr


def _link_binding(obj: Path, force: bool) -> None:
    import torch

    if not force and BINDING.exists() and BINDING.stat().st_mtime >= obj.stat().st_mtime:
        return
    libraries = Path(torch.__file__).resolve().parent / "lib"
    cmd = ["g++", "-shared", str(obj), "-o", str(BINDING), f"-L{LIBRARY.parent}",
           f"-l:{LIBRARY.name}", "-Wl,-rpath,$ORIGIN", f"-L{libraries}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")


def build(force: bool = False, jobs: int | None = None, verbose: bool = False,
          extra: list[str] | None = None) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    jobs = jobs or min(len(sources), os.cpu_count() or 4)
    lacks = binding_lacks()
    with ThreadPoolExecutor(max_workers=jobs + 1) as pool:
        binding = None if lacks else pool.submit(_compile_binding, force)
        results = list(pool.map(lambda s: _compile(s, force, extra or []), sources))
    objects = [obj for obj, _ in results]
    if verbose:
        for _, log in results:
            if log.strip():
                print(log, file=sys.stderr)
    newest = max(o.stat().st_mtime for o in objects)
    if force or not LIBRARY.exists() or LIBRARY.stat().st_mtime < newest:
        cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *map(str, objects),
               "-o", str(LIBRARY)]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")
    if binding is None:
        print(f"{BINDING.name} is not built, the 8-bit feed-forward operators have no Python side: {lacks}",
              file=sys.stderr)
    else:
        _link_binding(binding.result()[0], force)
    return LIBRARY


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--jobs", type=int, default=None)
    parser.add_argument("--verbose", action="store_true", help="print ptxas output")
    parser.add_argument("--ptxas-info", action="store_true", help="add -Xptxas -v")
    args = parser.parse_args()
    extra = ["-Xptxas", "-v"] if args.ptxas_info else []
    lib = build(force=args.force or args.ptxas_info, jobs=args.jobs,
                verbose=args.verbose or args.ptxas_info, extra=extra)
    print(lib)


if __name__ == "__main__":
    main()
