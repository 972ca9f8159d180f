"""Build the CUDA library in-tree for sm_100a.

    python -m atomflow_b200.build          # -> atomflow_b200/libatomflow_b200.so

nvcc cross-compiles without a GPU, so this runs on any machine with CUDA 12.8+.
The shared CUDA runtime is linked so the library shares the process's current
device and streams with any other CUDA user in the process (e.g. PyTorch).
"""
import importlib.metadata
import importlib.util
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libatomflow_b200.so"
CLI = PKG / "af_generate"        # the C++ greedy-decode driver on the C ABI
EXT = PKG / "_torch_ops.so"      # the paged operators for torch tensors (needs torch's headers)
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-cudart", "shared"]


def sources():
    return sorted(CSRC.glob("*.cu"))


def public_headers():
    return sorted((ROOT / "include").glob("*.h"))


def ext_source():
    return CSRC / "af_torch.cpp"


def headers():
    programs = [p for p in sorted(CSRC.glob("*.cpp")) if p != ext_source()]
    return sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + programs + public_headers()


def torch_root():
    """Where a torch built for CUDA is installed; None: nowhere, and the torch module is not built."""
    spec = importlib.util.find_spec("torch")
    root = Path(spec.origin).parent if spec is not None and spec.origin else None
    return root if root is not None and (root / "lib" / "libc10_cuda.so").exists() else None


def torch_version() -> str:
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:   # a torch on the path that no package manager put there
        return str(torch_root())


def ext_key() -> str:
    """What the torch module fits besides its sources: this torch, this Python."""
    return f"torch {torch_version()}, {sysconfig.get_config_var('SOABI')}"


def ext_stamp() -> Path:
    """Holds the ext_key of the module that was built last."""
    return PKG / "_build" / "torch_ops.txt"


def newer(target: Path, inputs) -> bool:
    return target.exists() and all(p.stat().st_mtime <= target.stat().st_mtime for p in inputs)


def lib_up_to_date() -> bool:
    return all(newer(t, sources() + headers()) for t in (LIB, CLI))


def ext_up_to_date() -> bool:
    if torch_root() is None:
        return True
    return (newer(EXT, [ext_source()] + public_headers()) and ext_stamp().exists() and
            ext_stamp().read_text() == ext_key())


def up_to_date() -> bool:
    return lib_up_to_date() and ext_up_to_date()


# Translation units whose element-wise arithmetic must round exactly like the
# reference's kernels, which are built with --use_fast_math (flush-to-zero and
# the approximate exp / reciprocal / rsqrt forms): the decode-step kernels.
FAST_MATH = {"af_decode.cu"}


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or not lib_up_to_date():
        build_lib(verbose)
    if force or not ext_up_to_date():
        build_ext(verbose)
    return LIB


def build_lib(verbose: bool = False) -> None:
    """The library and the C++ program on it."""
    nvcc = os.environ.get("NVCC", "nvcc")
    tmp = LIB.with_suffix(".so.tmp")
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)
    objs = []
    for src in sources():
        obj = objdir / (src.stem + ".o")
        extra = ["--use_fast_math"] if src.name in FAST_MATH else []
        cmd = [nvcc, *ARCH, *FLAGS, *extra, "-c", "-I", str(ROOT / "include"), "-o", str(obj), str(src)]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True, cwd=str(PKG))
        objs.append(str(obj))
    cmd = [nvcc, *ARCH, "-shared", "-cudart", "shared", "-o", str(tmp), *objs]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=str(PKG))
    os.replace(tmp, LIB)
    cmd = [nvcc, *ARCH, "-O2", "-std=c++17", "-I", str(ROOT / "include"), "-o", str(CLI),
           str(CSRC / "af_generate.cpp"), "-L", str(PKG), "-latomflow_b200", "-cudart", "shared",
           "-Xlinker", "-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=str(PKG))


def build_ext(verbose: bool = False) -> None:
    """The torch module over the C ABI; skipped where no torch built for CUDA is (the library itself does not need it)."""
    root = torch_root()
    if root is None:
        print("no torch built for CUDA: _torch_ops.so is not built", file=sys.stderr)
        return
    import torch
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    tmp = EXT.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(ROOT / "include"), "-isystem", str(root / "include"),
           "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", str(cuda / "include"), "-isystem", sysconfig.get_paths()["include"],
           "-o", str(tmp), str(CSRC / "af_torch.cpp"), "-L", str(PKG), "-latomflow_b200",
           "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=str(PKG))
    os.replace(tmp, EXT)
    ext_stamp().parent.mkdir(exist_ok=True)
    ext_stamp().write_text(ext_key())


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
