"""The build's own logic, without compiling anything."""
import sys

from fasterllama_b200 import build as B


def test_what_needs_no_torch_is_built_without_it(monkeypatch):
    done = []
    for name in ("build_cuda", "build_oracle", "build_reference", "build_e2e_variants"):
        monkeypatch.setattr(B, name, lambda *a, name=name, **k: done.append(name))
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises
    B.build_all()
    assert sorted(done) == ["build_cuda", "build_e2e_variants", "build_oracle", "build_reference"]
