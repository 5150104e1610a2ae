"""The native binding is built for one torch and Python, and the library works without it."""
from __future__ import annotations

import importlib.util
import sys
import warnings
from pathlib import Path

import pytest
import torch

from kernels import _lib
from test_serving_refusals_cpu import append_args, attention_args, verify_args

BUILD = Path(__file__).resolve().parents[1] / "simsd-release_b200" / "build.py"


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with an up-to-date library and a binding of its own under tmp_path; `calls` are its compiler runs."""
    spec = importlib.util.spec_from_file_location("simsd_build", BUILD)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    calls = []

    def run(cmds, verbose):
        calls.append(cmds)
        for c in cmds:
            Path(c[c.index("-o") + 1]).write_text("")

    monkeypatch.setattr(m, "OUT", tmp_path / "lib.so")
    monkeypatch.setattr(m, "BINDING", tmp_path / "_binding.so")
    monkeypatch.setattr(m, "OBJ", tmp_path)
    monkeypatch.setattr(m, "STAMP", tmp_path / "binding.stamp", raising=False)
    monkeypatch.setattr(m, "run", run)
    m.OUT.write_text("")
    m.calls = calls
    return m


def test_binding_of_another_torch_is_built_anew(build):
    build.build()
    assert len(build.calls) == 1 and any("SIMSD_BUILT_FOR" in a and torch.__version__ in a for a in build.calls[0][0])
    build.build()
    assert len(build.calls) == 1
    build.STAMP.write_text(build.STAMP.read_text().replace(str(torch.__version__), "1.0"))
    build.build()
    assert len(build.calls) == 2


@pytest.mark.parametrize("error", [RuntimeError("no headers"), FileNotFoundError("no compiler")])
def test_library_builds_without_the_binding(build, monkeypatch, capsys, error):
    build.BINDING.write_text("an older one")

    def run(cmds, verbose):
        raise error

    monkeypatch.setattr(build, "run", run)
    assert build.build() == build.OUT and build.OUT.exists()
    assert not build.BINDING.exists()                      # an older one is not used in its place
    assert str(error) in capsys.readouterr().err


def test_library_builds_without_torch(build, monkeypatch, capsys):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    assert build.build() == build.OUT and not build.calls and not build.BINDING.exists()
    assert "torch is not installed" in capsys.readouterr().err


def refuse_all():
    for f, args in ((_paged().paged_append, append_args()), (_paged().paged_attention, attention_args()),
                    (_verify().speculative_verify, verify_args())):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            f(**args)


def _paged():
    from kernels import paged_cache
    return paged_cache


def _verify():
    from kernels import spec_verify
    return spec_verify


def test_a_missing_binding_leaves_ctypes(monkeypatch):
    import kernels
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.delattr(kernels, "_binding", raising=False)
    monkeypatch.setitem(sys.modules, "kernels._binding", None)
    with pytest.warns(RuntimeWarning, match="through ctypes"):
        refuse_all()
    with warnings.catch_warnings():
        warnings.simplefilter("error")                     # said once
        refuse_all()
    monkeypatch.setattr(_lib, "_STREAM_SCRATCH", {})
    monkeypatch.setattr(_lib, "_WORKSPACES", {})
    _lib.clear_device_error(torch.device("cuda", 0))


def test_a_binding_of_another_torch_is_not_called(monkeypatch):
    import kernels

    class Other:
        built_for = "torch 1.0, Python 3.8"

        def __getattr__(self, name):
            raise AssertionError(name)

    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(kernels, "_binding", Other(), raising=False)
    monkeypatch.setitem(sys.modules, "kernels._binding", Other())
    with pytest.warns(RuntimeWarning, match="torch 1.0"):
        refuse_all()


def test_this_binding_is_of_this_torch():
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert _lib.binding().built_for == "torch %s, Python %d.%d" % (torch.__version__, *sys.version_info[:2])
