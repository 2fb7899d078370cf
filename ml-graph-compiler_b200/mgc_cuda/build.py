"""Build libmgc_cuda.so with nvcc for sm_100a, in tree.

The counterpart of the reference's C build driver (``codegen/build.py:129-209``): the compiler is
``$MGC_NVCC``, else ``nvcc`` on the PATH, else ``/usr/local/cuda/bin/nvcc``; the library is
rebuilt only when the hash of the sources and flags changes (the key is stored next to the
library), and written atomically. Unlike the C backend there is one library for every model:
a model is data (a launch list and a weights blob), not generated source. The paged-cache operators'
torch binding is a second, small module (``build_binding``).
"""

from __future__ import annotations

import hashlib
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

from mgc_cuda._errors import CodegenError

PACKAGE_DIR = Path(__file__).resolve().parent
SRC_DIR = PACKAGE_DIR.parent / "csrc"
INCLUDE_DIR = PACKAGE_DIR.parents[1] / "include"
LIB_DIR = PACKAGE_DIR / "lib"
LIB_NAME = "libmgc_cuda.so"
ARCH = os.environ.get("MGC_CUDA_ARCH", "sm_100a")


def find_nvcc() -> str:
    for cand in (os.environ.get("MGC_NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise CodegenError("nvcc not found (set MGC_NVCC)")


def nvcc_flags() -> list[str]:
    arch = ARCH.replace("sm_", "")
    return [
        "-O3",
        "-std=c++17",
        "-lineinfo",
        f"-gencode=arch=compute_{arch},code=sm_{arch}",
        "-Xcompiler=-fPIC,-O3,-Wall,-Wno-unused-function",
        "-shared",
        "--expt-relaxed-constexpr",
        f"-I{INCLUDE_DIR}",
        f"-I{SRC_DIR}",
    ]


def sources() -> list[Path]:
    return sorted([*SRC_DIR.glob("*.cu"), *SRC_DIR.glob("*.cuh"), *INCLUDE_DIR.glob("*.h")])


def binding_path() -> Path:
    """The torch binding of the paged-cache operators, a Python extension module."""
    return LIB_DIR / "_mgc_paged.so"


def _placeless(flags: list[str]) -> list[str]:
    """The flags without include paths: a tree that moved, sources unchanged, is still built."""
    return [f for f in flags if not f.startswith("-I")]


def source_key(flags: list[str]) -> str:
    flags = _placeless(flags)
    h = hashlib.sha256()
    for path in sources():
        h.update(path.name.encode())
        h.update(path.read_bytes())
    for f in flags:
        h.update(f.encode())
    return h.hexdigest()[:20]


def library_path() -> Path:
    return LIB_DIR / LIB_NAME


def _object_key(source: Path, flags: list[str]) -> str:
    """Key of one source file's object: its text, that of every header it includes, the flags."""
    seen: dict[Path, bytes] = {}
    todo = [source]
    while todo:
        path = todo.pop()
        if path in seen:
            continue
        seen[path] = path.read_bytes()
        for name in re.findall(rb'^\s*#include\s+"([^"]+)"', seen[path], flags=re.M):
            todo += [d / name.decode() for d in (SRC_DIR, INCLUDE_DIR) if (d / name.decode()).exists()]
    h = hashlib.sha256(" ".join(_placeless(flags)).encode())
    for path in sorted(seen):
        h.update(path.name.encode() + seen[path])
    return h.hexdigest()[:20]


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    proc = subprocess.run(cmd, capture_output=True, text=True, check=False)
    if proc.returncode != 0:
        raise CodegenError(f"{Path(cmd[0]).name} failed:\n{' '.join(cmd)}\n{proc.stderr[-6000:]}")
    if verbose and proc.stderr:
        print(proc.stderr[-6000:])


def _compile(source: Path, flags: list[str], force: bool, verbose: bool) -> Path:
    """The object of one source file, compiled if its key changed."""
    obj = LIB_DIR / f"{source.stem}.o"
    stamp = LIB_DIR / f"{source.stem}.o.key"
    key = _object_key(source, flags)
    if not force and obj.exists() and stamp.exists() and stamp.read_text().strip() == key:
        return obj
    tmp = obj.with_name(f"{obj.name}.tmp{os.getpid()}")
    _run([find_nvcc(), *(f for f in flags if f != "-shared"), "-c", str(source), "-o", str(tmp)], verbose)
    tmp.replace(obj)
    stamp.write_text(key + "\n")
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if the sources changed (its source files side by side); return its path."""
    flags = nvcc_flags()
    key = source_key(flags)
    lib = library_path()
    stamp = lib.with_suffix(".key")
    if not force and lib.exists() and stamp.exists() and stamp.read_text().strip() == key:
        return lib
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    units = sorted(SRC_DIR.glob("*.cu"))
    with ThreadPoolExecutor(max_workers=len(units)) as pool:
        objects = list(pool.map(lambda u: _compile(u, flags, force, verbose), units))
    tmp = lib.with_name(f"{LIB_NAME}.tmp{os.getpid()}")
    _run([find_nvcc(), *flags, *map(str, objects), "-o", str(tmp)], verbose)
    tmp.replace(lib)
    stamp.write_text(key + "\n")
    return lib


def _binding_flags() -> list[str]:
    import torch

    return ["-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]


def binding_key() -> str:
    """Key of the torch binding: its source and the header, the flags, torch's and Python's versions."""
    import sysconfig

    import torch

    return _object_key(SRC_DIR / "paged_torch.cpp", [*_binding_flags(), torch.__version__, sysconfig.get_python_version()])


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile the torch binding (csrc/paged_torch.cpp, host code) if it, the header or torch changed."""
    source, out = SRC_DIR / "paged_torch.cpp", binding_path()
    stamp, key = out.with_suffix(".key"), binding_key()
    if not force and out.exists() and stamp.exists() and stamp.read_text().strip() == key:
        return out
    import sysconfig

    from torch.utils import cpp_extension

    include = [*cpp_extension.include_paths(), sysconfig.get_path("include"), str(INCLUDE_DIR),
               str(Path(find_nvcc()).resolve().parents[1] / "include")]
    libs = cpp_extension.library_paths()
    flags = [*_binding_flags(), *(f"-I{p}" for p in include)]
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = out.with_name(f"{out.name}.tmp{os.getpid()}")
    cxx = os.environ.get("MGC_CXX") or shutil.which("g++") or "g++"
    _run([cxx, *flags, str(source), "-o", str(tmp), *(f"-L{p}" for p in libs), *(f"-Wl,-rpath,{p}" for p in libs),
          "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"], verbose)
    tmp.replace(out)
    stamp.write_text(key + "\n")
    return out


if __name__ == "__main__":
    print(build(force=True, verbose=True))
    print(build_binding(force=True, verbose=True))
