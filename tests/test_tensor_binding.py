"""The compiled binding belongs to the environment that it was built in (CPU)."""

from __future__ import annotations

import importlib.util
import os
import sys
from pathlib import Path

import pytest

from tklab import _tensors

SCRIPT = Path(__file__).resolve().parents[1] / "triton-kernel-lab_b200" / "build_native.py"
OTHER = "torch 1.0, cxx11 abi 0, cuda 9.0, cpython-36"


def library(stamp: str | None) -> bytes:
    """What stands in for an extension: bytes, with a stamp among them."""
    return b"\x7fELF\0\1" + (b"" if stamp is None else (_tensors.STAMP_MARK + stamp).encode() + b"\0") + b"\2\3"


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """The build script with an extension of its own; the compiler is only recorded."""
    spec = importlib.util.spec_from_file_location("build_native_copy", SCRIPT)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "BINDING_PATH", tmp_path / module.BINDING_PATH.name)
    module.ran = []

    def run(cmd, verbose):
        module.ran.append(cmd)
        (define,) = (arg for arg in cmd if arg.startswith("-DTKLAB_STAMP="))
        text = define.partition("=")[2].strip('"')
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"\x7fELF" + text.encode() + b"\0")
        return ""

    monkeypatch.setattr(module, "_run", run)
    return module


def test_rebuilt_for_another_environment(builder) -> None:
    for stamp in (None, OTHER, _tensors.binding_stamp() + "x"):
        builder.ran.clear()
        builder.BINDING_PATH.write_bytes(library(stamp))
        builder._build_binding(False, False)
        assert len(builder.ran) == 1 and _tensors.stamp_of(builder.BINDING_PATH) == _tensors.binding_stamp()
        builder._build_binding(False, False)
        assert len(builder.ran) == 1  # up to date
    os.utime(builder.BINDING_PATH, (0, 0))  # older than its source
    builder._build_binding(False, False)
    assert len(builder.ran) == 2


@pytest.mark.parametrize("stamp", [None, OTHER])
def test_not_loaded_in_another_environment(tmp_path, monkeypatch, stamp: str | None) -> None:
    path = tmp_path / _tensors.BINDING_PATH.name
    path.write_bytes(library(stamp))
    monkeypatch.setattr(_tensors, "BINDING_PATH", path)
    monkeypatch.delitem(sys.modules, "_tklab_tensors", raising=False)
    with pytest.raises(RuntimeError, match="was built for"):
        _tensors.load()


def test_the_built_extension_is_for_this_environment() -> None:
    assert _tensors.stamp_of(_tensors.BINDING_PATH) == _tensors.binding_stamp()
    _tensors.load()
