"""What the build makes where torch is missing or has changed; no compiler runs here."""
from __future__ import annotations

import pytest


@pytest.fixture
def build(monkeypatch, tmp_path):
    """The build module with its outputs in a folder of the test's and its commands collected."""
    from ffn_residual_mesh_b200 import build as b
    monkeypatch.setattr(b, "BIND", tmp_path / "bind.so")
    monkeypatch.setattr(b, "BIND_STAMP", tmp_path / "bind.stamp")
    monkeypatch.setattr(b, "LIB", tmp_path / "lib.so")
    monkeypatch.setattr(b, "BIN_DIR", tmp_path)
    calls = []

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        calls.append(out.rsplit("/", 1)[1])
        open(out, "w").close()

    monkeypatch.setattr(b.subprocess, "run", run)
    monkeypatch.setattr(b, "stale", lambda target=b.LIB, deps=None: not target.exists())
    b.LIB.touch()
    b.calls = calls
    yield b
    del b.calls


def test_library_and_runners_need_no_torch(build, monkeypatch, capsys):
    def missing(name):
        raise build.metadata.PackageNotFoundError(name)
    monkeypatch.setattr(build.metadata, "version", missing)
    build.build()
    assert build.calls == build.RUNNERS and "no torch" in capsys.readouterr().err


def test_binding_needs_torch_with_cuda(build, monkeypatch, capsys):
    import torch
    monkeypatch.setattr(torch.version, "cuda", None)
    build.build()
    assert build.calls == build.RUNNERS and "without CUDA" in capsys.readouterr().err


def test_binding_follows_torch_and_python(build, monkeypatch):
    build.build(runners=False)
    build.build(runners=False)
    assert build.calls == ["bind.so"]
    monkeypatch.setattr(build.metadata, "version", lambda name: "99.0")
    build.build(runners=False)
    build.build(runners=False)
    assert build.calls == ["bind.so"] * 2 and "torch 99.0" in build.BIND_STAMP.read_text()
    build.BIND.unlink()
    assert build.build_binding() == build.BIND and build.calls == ["bind.so"] * 3
