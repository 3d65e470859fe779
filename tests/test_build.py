"""The build's own logic, without compiling anything."""
import os
import subprocess
import sys

import torch

from fasterllama_b200 import build as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_what_needs_no_torch_is_built_without_it(monkeypatch):
    done = []
    for name in ("build_cuda", "build_oracle", "build_reference", "build_e2e_variants"):
        monkeypatch.setattr(B, name, lambda *a, name=name, **k: done.append(name))
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises
    B.build_all()
    assert sorted(done) == ["build_cuda", "build_e2e_variants", "build_oracle", "build_reference"]


def test_the_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    B.build_tensor_args()
    ran = []
    monkeypatch.setattr(B, "ARGS_STAMP", str(tmp_path / "stamp"))
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, **k: ran.append(cmd))
    B.build_tensor_args()  # no stamp: by whom it was built is not known
    assert len(ran) == 1
    B.build_tensor_args()
    assert len(ran) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    B.build_tensor_args()
    assert len(ran) == 2 and any("0.0.1" in x for x in ran[1])


def test_the_binding_refuses_another_torch():
    code = "import torch; torch.__version__ = '0.0.1'\ntry:\n    import fasterllama_b200._tensor_args\nexcept ImportError as e:\n    print(e)"
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, check=True).stdout
    assert "built for torch " + torch.__version__ in out and "0.0.1" in out
