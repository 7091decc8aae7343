"""The build without one of its parts."""

from __future__ import annotations

import shutil

import pytest

import __graft_entry__


@pytest.fixture
def build(monkeypatch, tmp_path):
    """The build module over one small source, into a folder of its own."""
    module = __graft_entry__._load_build_module()
    if shutil.which(module.HIPCC) is None:
        pytest.skip("needs hipcc")
    source = tmp_path / "small.cpp"
    source.write_text('extern "C" int small() { return 7; }\n')
    monkeypatch.setattr(module, "_sources", lambda: [source])
    monkeypatch.setattr(module, "BUILD_DIR", tmp_path / "_build")
    monkeypatch.setattr(module, "PKG_DIR", tmp_path)
    monkeypatch.setattr(module, "LIB_PATH", tmp_path / module.LIB_NAME)
    return module


def test_kernels_are_linked_where_the_binding_fails(build, monkeypatch):
    def fails():
        raise RuntimeError("no headers")

    monkeypatch.setattr(build, "_build_binding", fails)
    with pytest.raises(RuntimeError, match="no headers"):
        build.build()
    assert build.LIB_PATH.exists()


def test_the_binding_is_built_without_gxx(build, monkeypatch):
    commands = []

    def run(cmd, **kw):
        commands.append(cmd)
        return build.subprocess.CompletedProcess(cmd, 1, "", "not run")

    monkeypatch.delenv("CXX", raising=False)
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    monkeypatch.setattr(build.subprocess, "run", run)
    with pytest.raises(RuntimeError, match="not run"):
        build._build_binding()
    assert [c[0] for c in commands] == [build.HIPCC]


def test_a_binding_of_another_torch_is_refused(monkeypatch):
    import torch

    from mrun_pub_amd import _native as nat

    if not nat.LIB_PATH.exists():
        pytest.skip("library not built")
    assert nat.fast() is nat.fast()
    monkeypatch.setattr(nat, "_fast", None)
    monkeypatch.setattr(torch, "__version__", "1.0")
    with pytest.raises(RuntimeError, match="not 1.0"):
        nat.fast()
