"""Build step for libqgemv_b200.so (the sm_100a kernels + C-ABI) and the torch front end of
the paged cache operators -- run by
__graft_entry__.build() and, when the library is missing, by the package loader.
nvcc cross-compiles for sm_100a without a GPU."""

from __future__ import annotations

import os
import subprocess
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parents[1]          # local-ai-gpu-acceleration_b200/
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libqgemv_b200.so"
SOURCES = ["qg_gemv.cu", "qg_aux.cu", "qg_abi.cu", "qg_slice.cu", "qg_attn.cu", "qg_decode.cu",
           "qg_noalloc.cu", "qg_gemm_tc.cu", "qg_gguf.cu", "qg_gemv_batch.cu", "qg_paged_append.cu",
           "qg_paged_attn.cu", "qg_paged_evict.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_command(out: Path, extra: list[str] | None = None) -> list[str]:
    return [
        NVCC, *ARCH, "-lineinfo", "-O3", "-std=c++17", "-rdc=true",
        "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr",
        "--threads", "0", "-shared", "-o", str(out), *[str(CSRC / s) for s in SOURCES],
        "-lnccl",
        *(extra or []),
    ]


def up_to_date(out: Path = LIB_PATH) -> bool:
    if not out.exists():
        return False
    deps = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h"))
    deps.append(PKG_DIR.parent / "include" / "qgemv_b200.h")
    newest = max(p.stat().st_mtime for p in deps if p.exists())
    return out.stat().st_mtime >= newest


def scratch(out: Path) -> Path:
    """Where this process builds `out` before it takes its place: processes that build at the same
    time do not share it."""
    return out.with_name(f"{out.name}.{os.getpid()}.tmp")


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> Path:
    if not force and up_to_date():
        return LIB_PATH
    tmp = scratch(LIB_PATH)
    cmd = nvcc_command(tmp, extra)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        print(" ".join(cmd))
        print(res.stdout[-20000:])
        print(res.stderr[-20000:])
    if res.returncode != 0:
        tmp.unlink(missing_ok=True)
        raise RuntimeError(f"nvcc failed ({res.returncode}) building {LIB_PATH.name}")
    tmp.replace(LIB_PATH)
    return LIB_PATH


# The torch front end of the paged cache operators: a CPython module built with g++ against the
# torch that is installed; it holds no device code.
TORCH_SOURCE = CSRC / "qg_paged_torch.cpp"


def torch_path() -> Path:
    """The module of the installed torch and Python, by name: one that was compiled against the
    headers of another is never loaded."""
    import sysconfig

    import torch

    return PKG_DIR / f"qgemv_paged_torch.torch-{torch.__version__}.{sysconfig.get_config_var('SOABI')}.so"


def torch_command(out: Path) -> list[str]:
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = Path(NVCC).resolve().parents[1]
    include = [*cpp_extension.include_paths(), str(cuda / "include"), sysconfig.get_paths()["include"]]
    libs = Path(torch.__file__).parent / "lib"
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[f"-I{p}" for p in dict.fromkeys(include)], str(TORCH_SOURCE), "-o", str(out),
            f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]


def build_torch(force: bool = False) -> Path:
    header = PKG_DIR.parent / "include" / "qgemv_b200.h"
    newest = max(p.stat().st_mtime for p in (TORCH_SOURCE, header))
    out = torch_path()
    if not force and out.exists() and out.stat().st_mtime >= newest:
        return out
    tmp = scratch(out)
    cmd = torch_command(tmp)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        print(" ".join(cmd))
        print(res.stderr[-20000:])
        tmp.unlink(missing_ok=True)
        raise RuntimeError(f"g++ failed ({res.returncode}) building {out.name}")
    tmp.replace(out)
    return out


if __name__ == "__main__":
    import sys
    build(force=True, verbose=True, extra=sys.argv[1:])
    build_torch(force=True)
