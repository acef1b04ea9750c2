"""The library's sources as they lie in the tree."""

from __future__ import annotations

import subprocess

import pytest

from seoulkv_amd.build import CSRC, FLAGS, SOURCES, hipcc


@pytest.mark.parametrize("source", SOURCES)
def test_every_source_compiles(source):
    res = subprocess.run([hipcc(), *FLAGS, "-fsyntax-only", str(CSRC / source)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-4000:]
