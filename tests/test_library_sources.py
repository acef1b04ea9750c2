"""A library is that of the sources beside it, or is not loaded."""

from __future__ import annotations

import ctypes
import shutil

import pytest

from seoulkv_amd import _hip, build


@pytest.mark.parametrize("path", [build.LIB, _hip.TRACE_LIB_PATH, build.LIB.with_name("libseoulkv4_hip_asan.so")],
                         ids=lambda p: p.stem)
def test_built_libraries_are_of_these_sources(path):
    if not path.exists():
        if path == build.LIB:
            pytest.fail(f"{path} is not built")
        pytest.skip("not built")
    assert build.sources_id().encode() in path.read_bytes()


def test_a_library_of_other_sources_is_refused(tmp_path, monkeypatch):
    lib = ctypes.CDLL(str(build.LIB))
    assert _hip._of_these_sources(lib, build.LIB) is lib
    copy = tmp_path / "csrc"
    shutil.copytree(build.CSRC, copy)
    monkeypatch.setattr(build, "CSRC", copy)
    assert _hip._of_these_sources(lib, build.LIB) is lib
    with open(copy / "skv_tile.h", "a") as f:
        f.write("\n")
    monkeypatch.setattr(_hip, "_lib", None)
    monkeypatch.setattr(_hip, "_trace_lib", None)
    with pytest.raises(RuntimeError, match="other sources"):
        _hip.load_library()
    if _hip.TRACE_LIB_PATH.exists():
        with pytest.raises(RuntimeError, match="other sources"):
            _hip.load_trace_library()
    (copy / "skv_tile.h").unlink()
    with pytest.raises(RuntimeError, match="other sources"):
        _hip.load_library()


def test_a_library_without_a_hash_is_refused():
    class Old:
        pass

    with pytest.raises(RuntimeError, match="other sources"):
        _hip._of_these_sources(Old(), build.LIB)


def test_without_sources_nothing_is_compared(tmp_path, monkeypatch):
    monkeypatch.setattr(build, "CSRC", tmp_path / "none")
    lib = object()
    assert _hip._of_these_sources(lib, build.LIB) is lib


def test_a_failed_build_leaves_no_library(tmp_path, monkeypatch):
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "bad.hip").write_text("this is no source\n")
    monkeypatch.setattr(build, "CSRC", csrc)
    monkeypatch.setattr(build, "SOURCES", ["bad.hip"])
    monkeypatch.setattr(build, "LIB", tmp_path / "lib.so")
    for kind in ({}, {"trace": True}, {"sanitize_dir": tmp_path}):
        name = "libseoulkv4_hip_asan.so" if "sanitize_dir" in kind else "libseoulkv4_hip_trace.so" if kind else "lib.so"
        (tmp_path / name).write_bytes(b"an earlier build")
        with pytest.raises(RuntimeError, match="hipcc failed"):
            build.build(**kind)
        assert not (tmp_path / name).exists()
