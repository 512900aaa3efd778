"""Build recipe for the engine's C-ABI library (``libmoss_offload.so``) for gfx950.

Two steps, no torch extension machinery:

1. ``hipcc --genco --offload-arch=gfx950`` compiles each device source (``csrc/mo_device.hip``:
   pack/unpack/copy kernels; ``csrc/mo_gemm.hip``: int8 weight-only GEMMs; ``csrc/mo_fp8.hip``:
   8-bit floating-point quantizers and products; ``csrc/mo_rotary.hip``: rotary positions;
   ``csrc/mo_norm.hip``: norms; ``csrc/mo_gated.hip``: gated activations and activations in 8 bits;
   ``csrc/mo_adapters.hip``: low-rank adapters) into a standalone code object, embedded as a byte
   array.
2. ``g++`` compiles the host engine and launchers (``csrc/mo_engine.cpp``,
   ``csrc/mo_launch.cpp``, ...) with the embedded code objects into one shared library linked
   against the HIP runtime. The library loads its kernels with ``hipModuleLoadData`` on first
   use, so it registers no fat binary with the runtime.

Run ``python -m moss_offload.build`` from ``moss-image_amd/`` or call :func:`build`.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
SOURCE_ROOT = PACKAGE_DIR.parent
CSRC = SOURCE_ROOT / "csrc"
INCLUDE = SOURCE_ROOT.parent / "include"
BUILD_DIR = SOURCE_ROOT / "_build"
LIB_DIR = PACKAGE_DIR / "_lib"
LIB_PATH = LIB_DIR / "libmoss_offload.so"

# device source -> symbol of its embedded code object
DEVICE_SOURCES = {"mo_device.hip": "mo_device_code", "mo_gemm.hip": "mo_gemm_code", "mo_fp8.hip": "mo_fp8_code",
                  "mo_rotary.hip": "mo_rotary_code", "mo_norm.hip": "mo_norm_code", "mo_gated.hip": "mo_gated_code",
                  "mo_adapters.hip": "mo_adapters_code"}
HOST_SOURCES = ("mo_engine.cpp", "mo_launch.cpp", "mo_link.cpp", "mo_streamer.cpp", "mo_gemm.cpp", "mo_gradacc.cpp",
                "mo_fp8.cpp", "mo_rotary.cpp", "mo_norm.cpp", "mo_gated.cpp", "mo_adapters.cpp")

ARCH = "gfx950"

# Packed-FP32 instructions are disabled for all device code of this project.
DEVICE_FLAGS = [
    "--genco",
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-Wall",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
]

HOST_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__"]


def rocm_path() -> Path:
    return Path(os.environ.get("ROCM_PATH", "/opt/rocm"))


def hipcc() -> str:
    """Return the hipcc executable (ROCm's, or the one on PATH)."""

    candidate = rocm_path() / "bin" / "hipcc"
    if candidate.exists():
        return str(candidate)
    found = shutil.which("hipcc")
    if not found:
        raise RuntimeError("hipcc not found: the engine library cannot be built")
    return found


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"build step failed ({result.returncode}): {' '.join(cmd)}\n{result.stdout}\n{result.stderr}")
    if verbose and result.stderr.strip():
        print(result.stderr, file=sys.stderr)


def _blob_source(objects: dict[str, bytes]) -> str:
    parts = [
        "// Generated by moss_offload/build.py: the gfx950 code objects of csrc/*.hip.",
        "#include <stdint.h>",
    ]
    for symbol, code in objects.items():
        rows = [",".join(f"0x{b:02x}" for b in code[i : i + 16]) for i in range(0, len(code), 16)]
        body = ",\n".join(rows)
        parts.append(f'extern "C" __attribute__((aligned(4096))) const unsigned char {symbol}[{len(code)}] = {{\n{body}\n}};')
        parts.append(f'extern "C" const uint64_t {symbol}_size = {len(code)};')
    return "\n".join(parts) + "\n"


def build(verbose: bool = False) -> Path:
    """Compile the library into ``moss_offload/_lib`` and return its path.

    Always recompiles. The output is written to a temporary name and renamed, so a process
    that already loaded the previous library keeps a valid mapping.
    """

    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    objects = {}
    for source, symbol in DEVICE_SOURCES.items():
        code_object = BUILD_DIR / (Path(source).stem + ".co")
        _run([hipcc(), *DEVICE_FLAGS, f"-I{INCLUDE}", str(CSRC / source), "-o", str(code_object)], verbose)
        objects[symbol] = code_object.read_bytes()
    blob = BUILD_DIR / "mo_device_blob.cpp"
    blob.write_text(_blob_source(objects))
    tmp = LIB_DIR / f"libmoss_offload.so.tmp{os.getpid()}"
    rocm = rocm_path()
    cmd = ["g++", *HOST_FLAGS, f"-I{rocm / 'include'}", f"-I{INCLUDE}", "-o", str(tmp)]
    cmd += [str(CSRC / name) for name in HOST_SOURCES] + [str(blob)]
    cmd += [f"-L{rocm / 'lib'}", "-lamdhip64", "-lhsa-runtime64", "-lpthread", f"-Wl,-rpath,{rocm / 'lib'}"]
    try:
        _run(cmd, verbose)
    except Exception:
        tmp.unlink(missing_ok=True)
        raise
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
