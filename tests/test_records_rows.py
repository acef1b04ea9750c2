"""How the row tensors of the record cache's entry points may lie to each
other, without a GPU: over the HIP stub of ``records_stub_driver.c``."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from seoulkv_amd import _hip

HERE = Path(__file__).resolve().parent


def test_rows_that_share_memory(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not installed")
    exe, lib = tmp_path / "records_rows_driver", _hip.LIB_PATH
    subprocess.run(["gcc", "-std=gnu11", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__",
                    "-isystem", "/opt/rocm/include", "-I", str(HERE.parent / "include"), "-I", str(HERE),
                    str(HERE / "records_rows_driver.c"), "-o", str(exe), "-rdynamic", "-L", str(lib.parent),
                    "-lseoulkv4_hip", f"-Wl,-rpath,{lib.parent}", "-lm"], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, (res.returncode, res.stdout, res.stderr)
    assert "records rows driver ok" in res.stdout
