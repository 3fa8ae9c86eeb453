"""Build the native parts of carl_amd in-tree.

    python carl_amd/build.py          # engine + Python bindings
    python carl_amd/build.py --oracle # also the CPU oracle (test infrastructure)

(Run by path: importing the carl_amd package needs the extension built here.)

Outputs (next to this file):
  libcarl_amd.so   HIP engine and learner's operators for gfx950 + C-ABI
                   (include/carl_amd.h, include/carl_amd_ops.h)
  _carl*.so        pybind11 module exposing carl_amd._carl.Env
  _ops*.so         torch extension: the operators on torch tensors
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
ROCM = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
ARCH = os.environ.get("CARL_OFFLOAD_ARCH", "gfx950")

# -ffp-contract=off: every + - * / is one IEEE binary32 operation (the CPU
# model of the same physics is compiled the same way).  Packed FP32 math is
# disabled for all device code.
HIP_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
]

ENGINE_SOURCES = ["engine.hip", "arena.cpp", "adamw.hip", "attention.hip", "attention_f32.hip",
                  "attention_bf16.hip", "attention_f16.hip",
                  "ffn.hip", "ffn_f32.hip", "ffn_bf16.hip", "ffn_f16.hip", "actions.hip", "norm.hip", "int8.hip"]


def _run(cmd: list[str]) -> None:
    print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True, cwd=ROOT)


def engine_path() -> Path:
    return PKG / "libcarl_amd.so"


def binding_path(name: str = "_carl") -> Path:
    suffix = sysconfig.get_config_var("EXT_SUFFIX") or ".so"
    return PKG / f"{name}{suffix}"


def build_engine() -> Path:
    out = engine_path()
    hipcc = str(ROCM / "bin" / "hipcc")
    sources = [CSRC / name for name in ENGINE_SOURCES]
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(len(sources)) as pool:
        objects = [Path(tmp) / f"{src.name}.o" for src in sources]
        list(pool.map(lambda so: _run([hipcc, *HIP_FLAGS, "-c", str(so[0]), "-o", str(so[1])]), zip(sources, objects)))
        _run([hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(out), *map(str, objects)])
    return out


def build_binding() -> Path:
    import pybind11

    out = binding_path()
    py_inc = sysconfig.get_paths()["include"]
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
          "-D__HIP_PLATFORM_AMD__", f"-I{py_inc}", f"-I{pybind11.get_include()}",
          f"-I{ROCM / 'include'}", str(CSRC / "binding.cpp"),
          f"-L{PKG}", "-lcarl_amd", f"-L{ROCM / 'lib'}", "-lamdhip64",
          "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{ROCM / 'lib'}", "-o", str(out)])
    return out


def build_ops() -> Path:
    import torch
    from torch.utils import cpp_extension

    out = binding_path("_ops")
    py_inc = sysconfig.get_paths()["include"]
    torch_lib = Path(torch.__file__).resolve().parent / "lib"
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-attributes",
          "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", "-DTORCH_EXTENSION_NAME=_ops",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
          f"-I{py_inc}", *(f"-isystem{d}" for d in cpp_extension.include_paths()),
          f"-isystem{ROCM / 'include'}", str(CSRC / "ops_binding.cpp"),
          f"-L{PKG}", "-lcarl_amd", f"-L{torch_lib}", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10",
          "-lc10_hip", "-ltorch_python",
          "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{torch_lib}", f"-Wl,-rpath,{ROCM / 'lib'}", "-o", str(out)])
    return out


def build_oracle() -> Path:
    _run(["make", "-C", str(ROOT / "oracle"), "-B"])
    return ROOT / "oracle" / "liboracle.so"


def main(argv: list[str]) -> None:
    build_engine()
    build_binding()
    build_ops()
    if "--oracle" in argv:
        build_oracle()


if __name__ == "__main__":
    main(sys.argv[1:])
