"""Build libpagegauge_b200.so in-tree with nvcc for sm_100a, and the torch
binding of the rotary and 4-bit operators (_torch_ops.so) with the host
compiler.

    python -m pagegauge_b200.build [--force]
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sysconfig
from pathlib import Path

ROOT = Path(__file__).resolve().parent
CSRC = ROOT / "csrc"
INCLUDE = ROOT.parent / "include"
OUTPUT = ROOT / "libpagegauge_b200.so"
SOURCES = [CSRC / "pg_capi.cu"]
DEPENDS = SOURCES + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
BINDING = ROOT / "_torch_ops.so"
BINDING_SOURCE = CSRC / "pg_torch.cpp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    found = shutil.which("nvcc")
    if found:
        return found
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    return str(Path(cuda) / "bin" / "nvcc")


def command(output: Path = OUTPUT) -> list[str]:
    return [
        nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17",
        "-Xcompiler", "-fPIC", "-shared", "-Xptxas", "-v",
        "-I", str(INCLUDE),
        "-o", str(output), *map(str, SOURCES),
    ]


def binding_command(output: Path = BINDING) -> list[str]:
    import torch

    base = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return [
        os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
        "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
        "-I", str(INCLUDE), "-isystem", str(base / "include"),
        "-isystem", str(base / "include" / "torch" / "csrc" / "api" / "include"),
        "-isystem", sysconfig.get_paths()["include"], "-isystem", str(cuda / "include"),
        "-o", str(output), str(BINDING_SOURCE),
        f"-L{base / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
    ]


def up_to_date(output: Path = OUTPUT, depends=None) -> bool:
    if not output.is_file():
        return False
    built = output.stat().st_mtime
    return all(path.stat().st_mtime <= built for path in depends or DEPENDS)


def _compile(what: str, make, output: Path, verbose: bool) -> None:
    tmp = output.with_suffix(".so.tmp")
    proc = subprocess.run(make(tmp), capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{proc.stdout}\n{proc.stderr}")
    if verbose:
        print(proc.stderr)
    tmp.replace(output)


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or not up_to_date():
        _compile("nvcc", command, OUTPUT, verbose)
    if force or not up_to_date(BINDING, [BINDING_SOURCE, *INCLUDE.glob("*.h")]):
        _compile("the torch binding's compiler", binding_command, BINDING, verbose)
    return OUTPUT


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--force", action="store_true")
    args = parser.parse_args()
    print(build(force=args.force, verbose=True))


if __name__ == "__main__":
    main()
