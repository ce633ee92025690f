"""The module of autograd nodes is the one for the torch and the Python that run."""
import os
import sys

import pytest
import torch

from pointtransformerv3_b200 import _lib, build


def test_built_where_it_is_looked_for():
    build.build()
    path = _lib.nodes_path()
    assert path in build.nodes_command() and os.path.exists(path)
    assert _lib.nodes().__spec__.origin == path


@pytest.mark.parametrize("what", ["torch", "abi", "python"])
def test_one_for_another_torch_is_not_loaded(monkeypatch, what):
    build.build()
    present = _lib.nodes_path()
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "2.99.0")
    elif what == "abi":
        monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    else:
        monkeypatch.setattr(sys.implementation, "cache_tag", "cpython-399")
    monkeypatch.setattr(_lib, "_nodes", None)
    with pytest.raises(_lib.Ptv3Error, match="pointtransformerv3_b200.build"):
        _lib.nodes()
    # and a build is made for it
    assert _lib.nodes_path() != present and _lib.nodes_path() in build.nodes_command()
