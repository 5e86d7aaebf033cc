"""Build `libnt_b200.so` in-tree with nvcc for sm_100a.

The library is one translation unit (`csrc/nt_b200.cu` includes every kernel
family), compiled with `-gencode arch=compute_100a,code=sm_100a`.  It links only
the CUDA runtime; the TMA tensor-map encoder is fetched from the driver at run
time with `cudaGetDriverEntryPoint`, so no `-lcuda` is needed.

Beside it, a binding (`csrc/binding.cpp`, g++ against torch's headers) makes the
serving operators' calls in C++; without it they take their Python path.  It is
good for the Python and the torch that it was compiled against alone, and its
file's name says which.
"""

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
SOURCE_DIR = PACKAGE_DIR / "csrc"
LIBRARY = PACKAGE_DIR / "libnt_b200.so"
BINDING_SOURCE = SOURCE_DIR / "binding.cpp"
MAIN_SOURCE = SOURCE_DIR / "nt_b200.cu"
INCLUDE_DIR = PACKAGE_DIR.parent / "include"

NVCC_FLAGS = (
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    # function-local statics of templates (the per-device shared-memory
    # opt-in and occupancy caches) stay private to this library: as GNU
    # "unique" symbols a second build loaded into the same process would share
    # them and launch its kernels without their shared-memory opt-in
    "-Xcompiler",
    "-fno-gnu-unique",
    "-shared",
)


def find_nvcc() -> str:
    for candidate in (
        os.environ.get("NVCC"),
        shutil.which("nvcc"),
        os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc"),
    ):
        if candidate and os.path.isfile(candidate):
            return candidate
    raise FileNotFoundError("nvcc not found; set NVCC or CUDA_HOME")


def sources() -> list[Path]:
    """Files the library depends on, this one included (its compiler flags)."""
    return sorted(
        list(SOURCE_DIR.glob("*.cu"))
        + list(SOURCE_DIR.glob("*.cuh"))
        + list(INCLUDE_DIR.glob("*.h"))
        + [Path(__file__).resolve()]
    )


def _older(built: Path, paths) -> bool:
    return not built.is_file() or any(path.stat().st_mtime > built.stat().st_mtime for path in paths)


def binding_path() -> Path:
    """The binding's file for this Python and this torch."""
    import torch

    build = (getattr(torch.version, "git_version", None) or "")[:8]
    return PACKAGE_DIR / f"_binding.{sys.implementation.cache_tag}-torch-{torch.__version__}-{build}.so"


def binding_is_stale() -> bool:
    return _older(binding_path(), [BINDING_SOURCE, *INCLUDE_DIR.glob("*.h"), Path(__file__).resolve()])


def is_stale(library: Path = LIBRARY) -> bool:
    return _older(library, sources()) or binding_is_stale()


def build_binding(verbose: bool = False) -> Path:
    """Compile the C++ binding against the installed torch."""
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(find_nvcc()).resolve().parent.parent
    binding = binding_path()
    temporary = binding.with_name(f".{binding.name}.{os.getpid()}.tmp")
    command = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden"]
    command += [f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]
    command += [f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include", f"-I{cuda}/include"]
    command += [f"-I{sysconfig.get_paths()['include']}", "-o", str(temporary), str(BINDING_SOURCE), f"-L{root}/lib"]
    command += ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(command))
    try:
        subprocess.run(command, check=True)
        os.replace(temporary, binding)
    finally:
        if temporary.exists():
            temporary.unlink()
    return binding


def build_library(verbose: bool = False) -> Path:
    """Compile the library."""
    temporary = LIBRARY.with_name(f".{LIBRARY.name}.{os.getpid()}.tmp")
    command = [find_nvcc(), *NVCC_FLAGS]
    if verbose:
        command += ["-Xptxas", "-v"]
    command += ["-o", str(temporary), str(MAIN_SOURCE)]
    try:
        subprocess.run(command, check=True)
        os.replace(temporary, LIBRARY)
    finally:
        if temporary.exists():
            temporary.unlink()
    return LIBRARY


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library and the binding where they are missing or older than
    their sources.  A binding that cannot be compiled is a warning: its calls take
    their Python path."""
    if force or _older(LIBRARY, sources()):
        build_library(verbose)
    if force or binding_is_stale():
        try:
            build_binding(verbose)
        except (OSError, subprocess.CalledProcessError) as error:
            warnings.warn(f"the C++ binding of the serving calls was not built: {error}", stacklevel=2)
    return LIBRARY


if __name__ == "__main__":
    import sys

    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
