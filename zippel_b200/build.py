"""Builds the C-ABI shared library (CUDA kernels for sm_100a) in-tree with nvcc.

    python -m zippel_b200.build [--force] [--verbose]

Each ``csrc/*.cu`` is compiled to an object under ``csrc/_obj`` (skipped when newer than its
sources) and the objects are linked into ``zippel_b200/libzippel_b200.so``.  ``csrc/zp_rowwise_torch.cpp``,
functions on torch tensors over that library, becomes the extension module ``_rowwise`` beside it, for the
torch and Python that build it (and anew for others); where there is no torch for CUDA it is left out.
"""

from __future__ import annotations

import concurrent.futures
import importlib.metadata
import importlib.util
import os
import pathlib
import shutil
import subprocess
import sys

PKG = pathlib.Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = CSRC / "_obj"
LIB = PKG / "libzippel_b200.so"
TORCH_SOURCE = CSRC / "zp_rowwise_torch.cpp"      # the operators over rows, on torch tensors
ROWWISE = PKG / "_rowwise.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the kernels cannot be built")
    return exe


def _stale(target: pathlib.Path, deps: list[pathlib.Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build_library(force: bool = False, verbose: bool = False) -> pathlib.Path:
    OBJ.mkdir(exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted((ROOT / "include").glob("*.h"))
    sources = sorted(CSRC.glob("*.cu"))
    jobs = []
    torch_obj, made_for = OBJ / (TORCH_SOURCE.stem + ".o"), _made_for()
    if made_for is None:
        print("no torch for CUDA is installed: the functions on tensors (blocks/rowwise.py) are left out", file=sys.stderr)
    elif (force or _stale(torch_obj, [TORCH_SOURCE, ROOT / "include" / "zippel_b200.h"])
          or not _stamp().exists() or _stamp().read_text() != made_for):
        _stamp().unlink(missing_ok=True)
        jobs.append((TORCH_SOURCE, _torch_compile(torch_obj)))
    for src in sources:
        obj = OBJ / (src.stem + ".o")
        if force or _stale(obj, [src, *headers]):
            cmd = [nvcc(), *NVCC_FLAGS, "-I", str(ROOT / "include"), "-I", str(CSRC),
                   "-c", str(src), "-o", str(obj)]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append((src, cmd))

    def run(job):
        src, cmd = job
        res = subprocess.run(cmd, capture_output=True, text=True)
        return src, res

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        for src, res in ex.map(run, jobs):
            if verbose or res.returncode:
                sys.stderr.write(f"--- {src.name}\n{res.stdout}{res.stderr}\n")
            if res.returncode:
                raise RuntimeError(f"{'nvcc' if src.suffix == '.cu' else 'g++'} failed on {src.name}")
    objs = [OBJ / (s.stem + ".o") for s in sources]
    if force or _stale(LIB, objs):
        _link([nvcc(), "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"])
    if made_for is not None and (force or _stale(ROWWISE, [torch_obj]) or not _stamp().exists()):
        import torch
        libs = pathlib.Path(torch.__file__).parent / "lib"
        _link([_gxx(), "-shared", "-o", str(ROWWISE), str(torch_obj), "-L", str(libs), "-ltorch_python", "-ltorch_cuda",
               "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10", "-L", str(LIB.parent), "-lzippel_b200", "-Wl,-rpath,$ORIGIN"])
        _stamp().write_text(made_for)
    return LIB


def _made_for() -> str | None:
    """The torch and Python that an extension built now fits; None without a torch for CUDA."""
    torch = importlib.util.find_spec("torch")
    if torch is None or not (pathlib.Path(torch.origin).parent / "lib" / "libc10_cuda.so").exists():
        return None
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:          # (one that was not installed as a package)
        version = torch.origin
    return f"torch {version}, Python {sys.version}"


def _stamp() -> pathlib.Path:
    """Holds what the extension was last built for."""
    return OBJ / (TORCH_SOURCE.stem + ".for")


def _gxx() -> str:
    return shutil.which("g++") or "g++"


def _torch_compile(obj: pathlib.Path) -> list[str]:
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    includes = [*cpp_extension.include_paths(), str(pathlib.Path(nvcc()).resolve().parent.parent / "include"),
                sysconfig.get_paths()["include"], str(ROOT / "include")]
    return [_gxx(), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[a for i in includes for a in ("-isystem", i)], "-c", str(TORCH_SOURCE), "-o", str(obj)]


def _link(cmd: list[str]) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode:
        raise RuntimeError("link failed:\n" + res.stdout + res.stderr)


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
