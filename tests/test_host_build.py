"""The torch binding is tied to the torch and the Python that it was compiled against."""
import importlib.metadata

import pytest

from loractl_b200 import _build, _lib


def test_another_torch_means_a_build_of_its_own(monkeypatch):
    import torch

    _lib.ext()
    assert not _build.needs_build() and torch.__version__ in _build.torch_module().name
    version = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "2.0.0+cu118" if name == "torch" else version(name))
    monkeypatch.setattr(_lib, "_ext", None)
    assert _build.needs_build()
    with pytest.raises(RuntimeError, match="is missing"):
        _lib.ext()
