"""Build ``libseoulkv4_hip.so`` in-tree for gfx950 with hipcc.

Used by ``__graft_entry__.build()``; also runnable as
``python -m seoulkv_amd.build``.  The library is the only native artefact of
the package; ``seoulkv_amd._hip`` loads it from this directory.
"""

from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
HEADER = HERE.parent / "include" / "seoulkv4_hip.h"
LIB = HERE / "libseoulkv4_hip.so"
SOURCES = ["skv_runtime.hip", "skv_kernels.hip", "skv_dense.hip", "skv_cache.hip",
           "skv_rotary.hip", "skv_norm.hip", "skv_tree.hip", "skv_attend.hip", "skv_evict.hip"]
ARCH = os.environ.get("SKV_OFFLOAD_ARCH", "gfx950")

FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    # packed FP32 VALU forms are kept out of every device code object
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # leading scalar / pointer kernel arguments arrive in scalar registers at
    # dispatch (kernel argument preloading), so a kernel's first loads need
    # not wait for its argument block to be read from memory
    "-mllvm", "-amdgpu-kernarg-preload-count=16",
    "-Wall",
    "-Wno-unused-function",
    "-Wno-unused-variable",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found; the SeoulKV4 HIP library cannot be built")


# host code only: AddressSanitizer + UndefinedBehaviorSanitizer on the CPU
# side of the library (descriptor validation, mate and page tables, staging);
# the device code objects are built exactly as in the product library
SANITIZE_FLAGS = [
    "-Xarch_host", "-fsanitize=address",
    "-Xarch_host", "-fsanitize=undefined",
    "-Xarch_host", "-fno-sanitize-recover=all",
    "-Xarch_host", "-fno-omit-frame-pointer",
    "-g",
]


def sources_id() -> str:
    """What ``skv_sources()`` of a library built from this tree says: a hash of
    the sources, the header and the flags (but for the architecture)."""
    digest = hashlib.sha256(" ".join(f for f in FLAGS if not f.startswith("--offload-arch")).encode())
    for path in [*sorted(CSRC.iterdir()), HEADER]:
        if path.suffix in (".hip", ".h"):
            digest.update(path.name.encode() + b"\0" + path.read_bytes())
    return digest.hexdigest()[:32]


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"hipcc failed with exit code {res.returncode}")
    if verbose and res.stderr.strip():
        # hipcc's host pass reports the device-only target feature; harmless
        lines = [line for line in res.stderr.splitlines() if "packed-fp32-ops" not in line]
        if lines:
            print("\n".join(lines))


def build(verbose: bool = False, trace: bool = False, sanitize_dir: Path | None = None) -> Path:
    """Compile the library; ``trace`` builds the phase-timestamp variant
    ``libseoulkv4_hip_trace.so`` (development only) instead; ``sanitize_dir``
    builds ``libseoulkv4_hip_asan.so`` there, its host code instrumented with
    the address and undefined-behaviour sanitizers (tests only: a program
    that loads it must itself be linked with ``-fsanitize=address,undefined``
    by clang, which provides the runtime).  A library that is there goes first:
    a build that fails leaves none."""
    if sanitize_dir is not None:
        lib = Path(sanitize_dir) / "libseoulkv4_hip_asan.so"
    else:
        lib = LIB.with_name("libseoulkv4_hip_trace.so") if trace else LIB
    tmp = lib.with_suffix(".so.tmp")
    lib.unlink(missing_ok=True)
    extra = [f'-DSKV_SOURCES="{sources_id()}"']
    if trace:
        extra.append("-DSKV_TRACE")
    if sanitize_dir is not None:
        extra += SANITIZE_FLAGS
    with tempfile.TemporaryDirectory() as objects:
        outs = [str(Path(objects) / f"{Path(s).stem}.o") for s in SOURCES]
        compiles = [[hipcc(), *FLAGS, *extra, "-c", str(CSRC / s), "-o", o] for s, o in zip(SOURCES, outs)]
        # the largest sources take a minute: side by side
        with ThreadPoolExecutor(min(len(SOURCES), os.cpu_count() or 1, 8)) as pool:
            list(pool.map(lambda cmd: _run(cmd, verbose), compiles))
        _run([hipcc(), *FLAGS, *extra, "-shared", *outs, "-o", str(tmp)], verbose)
    os.replace(tmp, lib)
    return lib


if __name__ == "__main__":
    print(build(verbose=True, trace="--trace" in sys.argv[1:]))
