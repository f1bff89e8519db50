"""The build script's order of work, with the compilers replaced by a recorder."""
import sys
from pathlib import Path

import pytest

from dmuon_amd.csrc import build as b


@pytest.fixture
def recorded(monkeypatch, tmp_path):
    """Commands in their order; every one writes its output file."""
    commands = []

    def run(cmd, verbose):
        commands.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"")

    monkeypatch.setattr(b, "_run", run)
    monkeypatch.setattr(b, "_check_launch_stubs", lambda so: None)
    monkeypatch.setattr(b, "HERE", tmp_path)
    return commands


def test_the_library_is_built_without_torch(recorded, monkeypatch, tmp_path):
    monkeypatch.setitem(sys.modules, "torch", None)          # importing it raises
    assert b.build() == tmp_path / b.LIB_NAME
    assert (tmp_path / b.LIB_NAME).exists() and not (tmp_path / b.BINDING_NAME).exists()
    assert len(recorded) == len(b.SOURCES) + 1


def test_a_module_that_does_not_compile_leaves_the_library(recorded, monkeypatch, tmp_path):
    run = b._run

    def fail(cmd, verbose):
        if any(b.BINDING in part for part in cmd):
            raise RuntimeError("no module")
        run(cmd, verbose)

    monkeypatch.setattr(b, "_run", fail)
    with pytest.raises(RuntimeError, match="no module"):
        b.build()
    assert (tmp_path / b.LIB_NAME).exists() and not (tmp_path / b.BINDING_NAME).exists()


def test_both_are_built(recorded, tmp_path):
    b.build()
    assert (tmp_path / b.LIB_NAME).exists() and (tmp_path / b.BINDING_NAME).exists()
    assert len(recorded) == len(b.SOURCES) + 3


def test_a_module_of_another_torch_or_abi_is_refused(monkeypatch):
    import types

    import torch

    from dmuon_amd import _C
    ours = dict(abi_version=_C.ABI_VERSION, torch_version=str(torch.__version__))
    for other, text in ((dict(torch_version="2.9.1"), "torch 2.9.1"), (dict(abi_version=1), "version 1")):
        module = types.SimpleNamespace(**{**ours, **other})
        monkeypatch.setattr(_C, "_torch_ops", None)
        monkeypatch.setitem(sys.modules, "dmuon_amd.csrc._dmuon_torch", module)
        with pytest.raises(RuntimeError, match=text):
            _C.torch_ops()
        assert _C._torch_ops is None


def test_the_module_names_its_torch():
    import torch

    from dmuon_amd import _C
    assert _C.torch_ops().torch_version == str(torch.__version__)
