"""What build_all makes of the parts: the extension module of quantized.py is left out where torch is not installed, and its failure
keeps nothing else from being built."""
import importlib
import sysconfig

import pytest

import conftest


@pytest.fixture
def builder(monkeypatch):
    module = importlib.import_module(conftest.PKG_NAME + ".build")
    monkeypatch.setattr(module, "made", [], raising=False)
    for part in ("build_kernels", "build_host", "build_tools", "build_torch_ext"):
        monkeypatch.setattr(module, part, lambda *args, part=part: module.made.append(part) or part)
    return module


def test_every_part(builder):
    assert sorted(builder.build_all()) == ["build_host", "build_kernels", "build_tools", "build_torch_ext"]
    assert builder.made[0] == "build_kernels"  # (the others link it)


@pytest.mark.parametrize("missing", ["torch", "Python's headers"])
def test_without_what_the_extension_needs(builder, monkeypatch, capsys, tmp_path, missing):
    if missing == "torch":
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    else:
        paths = dict(sysconfig.get_paths(), include=str(tmp_path))
        monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: paths)
    assert builder.build_all() == ["build_kernels", "build_host", "build_tools"]
    assert missing in capsys.readouterr().out and "build_torch_ext" not in builder.made


def test_a_failing_extension_keeps_the_rest(builder, monkeypatch):
    def fail():
        raise RuntimeError("command failed: g++")

    monkeypatch.setattr(builder, "build_torch_ext", fail)
    with pytest.raises(RuntimeError, match="g\\+\\+"):
        builder.build_all()
    assert builder.made == ["build_kernels", "build_host", "build_tools"]
