"""Build the native library ``libpagedkv.so`` and the extension ``_int4_ops.so`` in-tree for sm_100a.

The library holds the C++ block ledger and the CUDA kernels behind the C ABI
declared in ``include/pagedkv.h``.  It is compiled with nvcc for
``arch=compute_100a,code=sm_100a`` and links the CUDA runtime statically, so
it loads (and the ledger runs) on machines without a GPU.  The extension binds
the 4-bit cache's operators of the library to torch tensors (host code only); where
torch with CUDA or Python's headers are missing, the library is built without it.

Usage: ``python -m pagedcore_b200.build [--force]``.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
REPO_ROOT = PACKAGE_DIR.parent
CSRC = PACKAGE_DIR / "csrc"
INCLUDE = REPO_ROOT / "include"
LIBRARY = PACKAGE_DIR / "libpagedkv.so"
BINDING = CSRC / "binding" / "int4_ops.cpp"
EXTENSION = PACKAGE_DIR / "_int4_ops.so"
EXTENSION_STAMP = PACKAGE_DIR / "_int4_ops.built_for"  # built_for() of the build that made it

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def sources() -> list[Path]:
    return sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cpp")])


def _inputs() -> list[Path]:
    return [*sources(), *CSRC.glob("*.h"), *CSRC.glob("*.cuh"), *INCLUDE.glob("*.h")]


def _library_up_to_date() -> bool:
    if not LIBRARY.exists():
        return False
    built = LIBRARY.stat().st_mtime
    return all(path.stat().st_mtime <= built for path in _inputs())


def built_for() -> str:
    """What a build of the extension is tied to: this Python's and this torch's binary interfaces."""
    import torch

    return f"{sysconfig.get_config_var('SOABI')}, torch {torch.__version__}, C++11 ABI {int(torch.compiled_with_cxx11_abi())}"


def extension_lacks() -> str | None:
    """What the extension's build needs and this machine has not, or None."""
    try:
        import torch
    except ImportError:
        return "torch"
    root = Path(torch.__file__).resolve().parent
    needed = {
        "Python's headers": Path(sysconfig.get_paths()["include"]) / "Python.h",
        "torch's headers": root / "include" / "ATen" / "ATen.h",
        "torch with CUDA": root / "lib" / "libtorch_cuda.so",
    }
    return next((name for name, path in needed.items() if not path.exists()), None)


def _extension_up_to_date() -> bool:
    if not EXTENSION.exists() or not EXTENSION_STAMP.exists() or EXTENSION_STAMP.read_text() != built_for():
        return False
    built = EXTENSION.stat().st_mtime
    return all(path.stat().st_mtime <= built for path in (BINDING, *INCLUDE.glob("*.h")))


def up_to_date() -> bool:
    return _library_up_to_date() and (extension_lacks() is not None or _extension_up_to_date())


def nvcc() -> str:
    found = shutil.which("nvcc")
    if found:
        return found
    default = Path("/usr/local/cuda/bin/nvcc")
    if default.exists():
        return str(default)
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libpagedkv.so")


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every source into ``libpagedkv.so``, then the extension (each skipped when up to date).

    The extension is left out, with a line on stderr, where what it needs is missing: only
    :mod:`pagedcore_b200.int4` is without it then.
    """
    if force or not _library_up_to_date():
        _build_library(verbose)
    lacks = extension_lacks()
    if lacks is not None:
        print(f"{EXTENSION.name} (the 4-bit cache's operators) is not built: {lacks} not found", file=sys.stderr)
    elif force or not _extension_up_to_date():
        _build_extension(verbose)
    return LIBRARY


def _build_library(verbose: bool) -> None:
    tmp = LIBRARY.with_suffix(".so.tmp")
    command = [
        nvcc(),
        *ARCH_FLAGS,
        "-O3",
        "-lineinfo",
        "-std=c++17",
        "-Xcompiler",
        "-fPIC,-O3",
        "-shared",
        "-cudart",
        "static",
        f"-I{INCLUDE}",
        f"-I{CSRC}",
        "-o",
        str(tmp),
        *[str(path) for path in sources()],
    ]
    if verbose:
        command.insert(1, "-Xptxas=-v")
    _run(command, tmp, LIBRARY, verbose)


def _build_extension(verbose: bool) -> None:
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = EXTENSION.with_suffix(".so.tmp")
    command = [
        os.environ.get("CXX", "g++"),
        "-O2",
        "-std=c++17",
        "-fPIC",
        "-shared",
        "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
        f'-DPKV_BUILT_FOR="{built_for()}"',
        f"-I{INCLUDE}",
        f"-I{root / 'include'}",
        f"-I{root / 'include' / 'torch' / 'csrc' / 'api' / 'include'}",
        f"-I{cuda / 'include'}",
        f"-I{sysconfig.get_paths()['include']}",
        str(BINDING),
        "-o",
        str(tmp),
        f"-L{root / 'lib'}",
        "-ltorch_python",
        "-ltorch_cuda",
        "-ltorch_cpu",
        "-ltorch",
        "-lc10",
        "-lc10_cuda",
        f"-L{PACKAGE_DIR}",
        f"-l:{LIBRARY.name}",
        "-Wl,-rpath,$ORIGIN",
    ]
    _run(command, tmp, EXTENSION, verbose)
    EXTENSION_STAMP.write_text(built_for())


def _run(command: list[str], tmp: Path, target: Path, verbose: bool) -> None:
    if verbose:
        print(" ".join(command), file=sys.stderr)
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"building {target.name} failed:\n{result.stdout}\n{result.stderr}")
    if verbose and result.stderr:
        print(result.stderr, file=sys.stderr)
    os.replace(tmp, target)


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
