"""Build the native pieces of leo_amd.

    python -m leo_amd.build            # libleo_hip.so (gfx950), its torch binding, the CPU oracle

libleo_hip.so holds the HIP kernels, the host runtime and the C-ABI of
include/leo_hip.h, include/leo_formats.h and include/leo_decode.h. It is built
in-tree (leo_amd/_lib/) so that it travels with the repository. Every HIP
translation unit is compiled with
-ffp-contract=off (the kernels must round exactly where Leo's CPU executor
rounds) and with packed-FP32 instructions disabled.
"""
from __future__ import annotations

import importlib.util
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

ROOT = pathlib.Path(__file__).resolve().parents[1]
CSRC = ROOT / "leo_amd" / "csrc"
LIB_DIR = ROOT / "leo_amd" / "_lib"
LIB = LIB_DIR / "libleo_hip.so"
BINDING = LIB_DIR / "leo_decode_binding.so"
BUILD = ROOT / "_build"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    f"-I{ROOT / 'include'}",
    f"-I{CSRC}",
]
CXX_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-pthread", "-ffp-contract=off", "-Wall", "-Wextra",
             f"-I{ROOT / 'include'}", f"-I{CSRC}"]


def _run(cmd):
    print("+ " + " ".join(str(c) for c in cmd), flush=True)
    subprocess.run([str(c) for c in cmd], check=True)


def build_library() -> pathlib.Path:
    BUILD.mkdir(exist_ok=True)
    LIB_DIR.mkdir(exist_ok=True)
    commands, objects = [], []
    for src in ("leo_kernels.hip", "leo_runtime.hip", "leo_q4.hip", "leo_answer.hip", "leo_q8.hip", "leo_beams.hip"):
        objects.append(BUILD / (src + ".o"))
        commands.append([HIPCC, *HIP_FLAGS, "-c", CSRC / src, "-o", objects[-1]])
    for src in ("host_model.cpp", "formats.cpp"):
        objects.append(BUILD / (pathlib.Path(src).stem + ".o"))
        commands.append([os.environ.get("CXX", "g++"), *CXX_FLAGS, "-c", CSRC / src, "-o", objects[-1]])
    with ThreadPoolExecutor(max_workers=len(commands)) as pool:   # one compiler process each
        list(pool.map(_run, commands))
    tmp = LIB.with_suffix(".so.tmp")
    _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-pthread", *objects, "-o", tmp])
    os.replace(tmp, LIB)
    return LIB


def build_binding() -> pathlib.Path:
    """The torch face of include/leo_decode.h: host code only, beside the library it calls."""
    import torch
    from torch.utils.cpp_extension import include_paths

    tmp, lib = BINDING.with_suffix(".so.tmp"), pathlib.Path(torch.__file__).parent / "lib"
    _run([os.environ.get("CXX", "g++"), *CXX_FLAGS, "-shared",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
          *(f"-isystem{path}" for path in (*include_paths(), sysconfig.get_paths()["include"])),
          CSRC / "decode_binding.cpp", "-o", tmp, f"-L{lib}", "-ltorch_python", "-ltorch_hip", "-ltorch_cpu", "-lc10",
          f"-L{LIB_DIR}", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"])
    os.replace(tmp, BINDING)
    return BINDING


def build_oracle() -> pathlib.Path:
    _run(["make", "-s", "-B", "-C", ROOT / "oracle"])
    return ROOT / "oracle" / "liboracle.so"


def main() -> int:
    subprocess.run([sys.executable, str(CSRC / "gen_abi.py"), "--check"], check=True)
    build_library()
    if importlib.util.find_spec("torch"):   # the step runtime does without
        build_binding()
    if shutil.which("make"):
        build_oracle()
    return 0


if __name__ == "__main__":
    sys.exit(main())
