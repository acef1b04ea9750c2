"""Index building needs no GPU: the package imports on a build of PyTorch
without one, as before it had operators of its own streams."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_the_package_imports_without_the_gpu_bindings():
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]: delattr(torch._C, name)\n"
            "import seoulkv_amd\n"
            "assert seoulkv_amd.SeoulKV4Index and seoulkv_amd.rotary\n")
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=180)
    assert res.returncode == 0, res.stderr
