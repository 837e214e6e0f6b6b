"""What the build makes of torch: without it the rest is built, and _ops.so follows
the torch that is installed."""
import importlib.metadata
import importlib.util

import pytest

from chpe_qwen_engine_b200 import build


def test_without_torch_the_rest_is_built(monkeypatch, capsys):
    for name in ("synth", "engine", "cli"):
        monkeypatch.setattr(build, "build_" + name, lambda force, name=name: name)
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setattr(build.subprocess, "run", lambda *a, **kw: pytest.fail("nothing to compile"))
    assert build.build_all(force=True) == ["synth", "engine", "cli"]
    assert "no torch" in capsys.readouterr().err


def test_a_torch_without_cuda_counts_as_none(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("torch", tmp_path / "__init__.py")
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec)
    assert build.build_ops() is None


def test_ops_follow_torch(monkeypatch, tmp_path):
    pytest.importorskip("torch")
    if not build._torch_tag():
        pytest.skip("a torch without CUDA")
    ran = []

    def run(cmd, check):
        ran.append(cmd)
        (tmp_path / "_ops.so").write_text("")
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "OPS", str(tmp_path / "_ops.so"))
    monkeypatch.setattr(build, "OPS_TAG", str(tmp_path / "x" / "_ops.tag"))
    for version, count in ((None, 1), (None, 1), ("0.0.1", 2), ("0.0.1", 2)):
        if version:
            monkeypatch.setattr(importlib.metadata, "version", lambda name: version)
        assert build.build_ops() == str(tmp_path / "_ops.so") and len(ran) == count
    assert build.build_ops(force=True) and len(ran) == 3
