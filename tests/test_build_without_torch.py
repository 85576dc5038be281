"""The library builds and loads where torch is missing, and the binding to torch is one for each torch."""
import importlib.metadata
import importlib.util

import pytest

from gptoss_b200 import capi


def test_the_library_needs_no_torch(monkeypatch):
    if capi.needs_build():
        capi.build()

    def version(name):
        raise importlib.metadata.PackageNotFoundError(name)

    ran = []
    monkeypatch.setattr(importlib.metadata, "version", version)
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None)
    monkeypatch.setattr(capi, "_nvcc", lambda args: ran.append(args) or "")
    monkeypatch.setattr(capi, "TORCH_LIB_PATH", capi._torch_lib_path())
    assert capi.TORCH_LIB_PATH is None
    assert not capi.needs_build()
    assert capi.build(force=True) == capi.LIB_PATH
    assert [a[a.index("-o") + 1] for a in ran] == [str(capi.LIB_PATH)]
    assert capi.load() is not None


def test_the_binding_is_named_after_the_torch_it_is_for(monkeypatch):
    paths = set()
    for v in ("2.11.0+cu128", "2.12.0", "2.12.1"):
        monkeypatch.setattr(importlib.metadata, "version", lambda name, v=v: v)
        paths.add(capi._torch_lib_path())
    assert len(paths) == 3
    monkeypatch.setattr(capi, "TORCH_LIB_PATH", capi.CSRC / "_serving_torch.of-another-torch.so")
    assert capi.needs_build()  # it has not been built


def test_the_torch_layer_says_that_its_binding_is_missing(monkeypatch):
    pytest.importorskip("torch")
    from gptoss_b200 import serving
    monkeypatch.setattr(serving, "_binding", None)
    for path in (None, capi.CSRC / "_serving_torch.of-another-torch.so"):
        monkeypatch.setattr(capi, "TORCH_LIB_PATH", path)
        with pytest.raises(RuntimeError):
            serving.route_experts(None, 1)
