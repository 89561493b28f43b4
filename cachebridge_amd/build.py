"""Build ``libcachebridge_hip.so`` in-tree with hipcc for gfx950.

    python -m cachebridge_amd.build
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
SOURCES = [PACKAGE / "csrc" / "cb_handoff.hip", PACKAGE / "csrc" / "cb_queries.hip"]
OUTPUT = PACKAGE / "libcachebridge_hip.so"
ARCH = os.environ.get("CACHEBRIDGE_OFFLOAD_ARCH", "gfx950")

FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # Keep the compiler from emitting packed fp32 VALU ops on this target.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
]


def hipcc() -> str:
    for candidate in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("hipcc not found")


def build_library(verbose: bool = False) -> Path:
    """Compile every HIP source (at the same time) and link the package's shared library."""
    tmp = OUTPUT.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory() as work:
        objects = [Path(work) / f"{source.stem}.o" for source in SOURCES]
        steps = [[[hipcc(), *FLAGS, "-c", str(source), "-o", str(obj)] for source, obj in zip(SOURCES, objects)],
                 [[hipcc(), *FLAGS, "-shared", *map(str, objects), "-o", str(tmp)]]]
        for commands in steps:
            running = [subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
                       for cmd in commands]
            output = [process.communicate()[0] for process in running]
            for cmd, process, text in zip(commands, running, output):
                if verbose or process.returncode:
                    sys.stderr.write(text)
                if process.returncode:
                    raise RuntimeError(f"hipcc failed ({process.returncode}): {' '.join(cmd)}")
    os.replace(tmp, OUTPUT)
    return OUTPUT


if __name__ == "__main__":
    print(build_library(verbose="-v" in sys.argv))
