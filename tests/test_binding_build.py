"""The native binding is built anew for another torch."""
import torch

from mlp_megakernel_b200 import _native, build


def test_another_torch_makes_it_stale(built_lib, monkeypatch):
    assert not build._binding_stale()
    assert _native.native().built_for == build.built_for()
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    assert build._binding_stale()
    monkeypatch.undo()
    assert not build._binding_stale()
