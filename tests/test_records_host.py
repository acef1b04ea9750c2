"""The record cache's host side without a GPU: what the C entry points refuse
(over a stub of the HIP runtime, ``records_stub_driver.c``), the angles of the
rotary table, what the Python layer refuses before it needs a device."""

from __future__ import annotations

import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from seoulkv_amd import RecordCache, RotaryTable, _hip, rotary
from seoulkv_amd.rope import _turns, scaled_frequencies

HERE = Path(__file__).resolve().parent


def test_entry_points_refuse_what_they_cannot_take(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not installed")
    exe, lib = tmp_path / "records_stub_driver", _hip.LIB_PATH
    subprocess.run(["gcc", "-std=gnu11", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__",
                    "-isystem", "/opt/rocm/include", "-I", str(HERE.parent / "include"),
                    str(HERE / "records_stub_driver.c"), "-o", str(exe), "-rdynamic", "-L", str(lib.parent),
                    "-lseoulkv4_hip", f"-Wl,-rpath,{lib.parent}", "-lm"], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, (res.returncode, res.stdout, res.stderr)
    assert "records stub driver ok" in res.stdout


@pytest.mark.parametrize("values", [[1.0, 0.5, 1e-6], [2 * math.pi, math.pi, -1.0], [1e-12, 100.0]])
def test_turns_are_the_angles(values):
    """2^-64 turns, rounded once: the fraction of a turn to double precision
    (2^-53 of the angle in turns, and the reduction's last digit)."""
    for x, t in zip(values, _turns(values).tolist()):
        fraction = t / 2.0**64
        off = (x / (2 * math.pi) - fraction) % 1.0
        assert min(off, 1 - off) <= abs(x) * 2.0**-52


def test_scaled_frequencies():
    plain, one = scaled_frequencies(8, 10000.0)
    assert plain == [10000.0 ** (-i / 4) for i in range(4)] and one == 1.0
    assert scaled_frequencies(8, 10000.0, ("linear", 4.0))[0] == [x / 4 for x in plain]
    ntk = scaled_frequencies(8, 10000.0, ("ntk", 4.0))[0]
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)  # the slowest pair is stretched by f
    yarn, scale = scaled_frequencies(128, 10000.0, ("yarn", 8.0, 4096))
    base = scaled_frequencies(128, 10000.0)[0]
    assert scale == pytest.approx(0.1 * math.log(8) + 1)
    turns = [4096 * x / (2 * math.pi) for x in base]
    for x, y, t in zip(base, yarn, turns):
        assert x / 8 * (1 - 1e-12) <= y <= x * (1 + 1e-12)
        if t > 36:
            assert y == x
        if t < 0.9:
            assert y == pytest.approx(x / 8)
    for bad in (("linear",), ("linear", 2.0, 3.0), ("yarn", 2.0), ("yarn", 2.0, 0.0), ("yarn", 2.0, 64, 1, 32),
                ("other", 2.0), ("linear", -1.0), ("ntk", math.inf)):
        with pytest.raises(ValueError):
            scaled_frequencies(8, 10000.0, bad)
    with pytest.raises(ValueError):
        scaled_frequencies(8, 1.0)


def test_the_python_layer_refuses_before_a_device():
    for kwargs in ({"rotary_dim": 7}, {"rotary_dim": 0}, {"rotary_dim": 1026}, {"rotary_dim": 8, "layout": "other"},
                   {"rotary_dim": 8, "device": "cpu"}):
        with pytest.raises(ValueError):
            RotaryTable(**kwargs)
    for kwargs in ({"inverse_frequencies": [1.0]}, {"inverse_frequencies": [1.0, math.nan]}, {"scale": math.inf},
                   {"inverse_frequencies": [1.0, 2.0], "scaling": ("linear", 2.0)}):
        with pytest.raises(ValueError):
            RotaryTable(4, **kwargs)
    with pytest.raises(TypeError):
        rotary(torch.zeros(1, 1, 4), torch.zeros(1), None)
    for records in (torch.zeros(1, 4, 16, 512, dtype=torch.uint8), torch.zeros(1, 4, 16, 512), None):
        with pytest.raises(ValueError):
            RecordCache(records, [0])
    for args in ((0, 16), (1025, 16), (1, 0), (1, (1 << 20) + 1), (1.0, 16)):
        with pytest.raises(ValueError):
            RecordCache.allocate(*args, device="cpu")
