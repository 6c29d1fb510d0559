"""Build recipe for the in-tree HIP library ``ascendflow_amd/libascendflow_amd.so``.

Every source under ``csrc/`` is compiled for gfx950 only, with packed-FP32
instruction selection switched off, and linked into one shared library that
exports the C ABI of ``include/ascendflow_amd.h``.
"""

from __future__ import annotations

import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
BUILD_DIR = PACKAGE / "_build"
LIBRARY = PACKAGE / "libascendflow_amd.so"
ARCH = "gfx950"

HIP_FLAGS = (
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    # A loop marked for unrolling that the compiler leaves as it is keeps its register arrays in memory.
    "-Werror=pass-failed",
    # gfx950 packed-FP32 forms are kept out of every kernel.
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    f"-I{ROOT / 'include'}",
)

# Device code of the other sources holds no NaNs of its own (masked scores are
# -inf, never NaN): without this, every fmaxf on a value the compiler cannot prove
# canonical (MFMA results, lane swaps) gets an extra v_max_f32 x, x to quiet
# signalling NaNs. Host code keeps IEEE NaN semantics (the launchers' argument checks).
NO_NAN_FLAGS = ("-Xarch_device", "-fno-honor-nans")
# Sources whose kernels pass NaNs of their inputs on.
NAN_SOURCES = ("quantized_cache", "rotary")


def hipcc() -> str:
    found = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(found).exists():
        raise RuntimeError("hipcc not found: the ROCm toolchain is required to build")
    return found


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


def _compile(src: Path) -> Path:
    obj = BUILD_DIR / (src.stem + ".o")
    flags = HIP_FLAGS if src.stem in NAN_SOURCES else HIP_FLAGS + NO_NAN_FLAGS
    cmd = [hipcc(), *flags, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{proc.stderr}")
    return obj


def build(verbose: bool = False) -> Path:
    """Compile every HIP source and link the shared library; returns its path."""
    BUILD_DIR.mkdir(exist_ok=True)
    srcs = sources()
    workers = max(1, min(len(srcs), int(os.environ.get("MAX_JOBS", "8"))))
    with ThreadPoolExecutor(workers) as pool:
        objects = list(pool.map(_compile, srcs))
    tmp = LIBRARY.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objects), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, LIBRARY)
    if verbose:
        print(f"built {LIBRARY} from {[s.name for s in srcs]}")
    return LIBRARY


if __name__ == "__main__":
    build(verbose=True)
