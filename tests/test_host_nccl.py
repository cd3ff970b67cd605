"""Which NCCL a process gets."""

from types import SimpleNamespace

import pytest


@pytest.mark.parametrize("torch", [True, False])
def test_the_environments_nccl_is_loaded_for_torch_alone(monkeypatch, tmp_path, torch):
    """Without PyTorch nothing needs it, and the engine keeps the library that it was linked with."""
    from tynx_b200 import _native

    library = tmp_path / "nccl" / "lib" / "libnccl.so.2"
    library.parent.mkdir(parents=True)
    library.touch()
    specs = {"nvidia": SimpleNamespace(submodule_search_locations=[str(tmp_path)])}
    if torch:
        specs["torch"] = SimpleNamespace()
    loaded = []
    monkeypatch.setattr(_native.importlib.util, "find_spec", specs.get)
    monkeypatch.setattr(_native.C, "CDLL", loaded.append)
    _native._share_nccl()
    assert loaded == ([str(library)] if torch else [])
