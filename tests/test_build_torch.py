"""When the tensor module _hsg_torch is rebuilt."""
import os

import pytest
import torch

from hs_guard_b200 import build


@pytest.fixture(scope="module", autouse=True)
def built():
    build.build_torch()


def test_a_fresh_module_is_not_stale():
    assert not build.torch_stale()
    before = os.path.getmtime(build.TORCH_LIB)
    assert build.build_torch() == build.TORCH_LIB and os.path.getmtime(build.TORCH_LIB) == before


@pytest.mark.parametrize("name,value", [("__version__", "2.0.0+other"), ("__file__", "/elsewhere/torch/__init__.py")])
def test_another_torch_makes_it_stale(monkeypatch, name, value):
    monkeypatch.setattr(torch, name, value)
    assert build.torch_stale()


def test_a_missing_stamp_or_module_makes_it_stale(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "TORCH_STAMP", str(tmp_path / "none"))
    assert build.torch_stale()
    monkeypatch.undo()
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "none.so"))
    assert build.torch_stale()


def test_a_changed_source_makes_it_stale(monkeypatch, tmp_path):
    newer = tmp_path / "newer.cpp"
    newer.write_text("")
    later = os.path.getmtime(build.TORCH_LIB) + 10
    os.utime(newer, (later, later))
    monkeypatch.setattr(build, "TORCH_SRC", str(newer))
    assert build.torch_stale()
