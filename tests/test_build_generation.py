"""The build of the module over torch tensors: the other parts are built without
torch, and another torch rebuilds it."""
import os
import sys

from chimera_b200 import build as B


def test_a_build_without_torch_leaves_the_module_over_torch_out(monkeypatch, capsys):
    built = []
    for part in ("build_cuda", "build_hostrng", "build_host"):
        monkeypatch.setattr(B, part, lambda *a, part=part: built.append(part))
    monkeypatch.setitem(sys.modules, "torch", None)   # import torch raises ImportError
    B.build()
    assert built == ["build_cuda", "build_hostrng", "build_host"]
    assert "torch" in capsys.readouterr().out


def test_another_torch_rebuilds_the_module(monkeypatch, tmp_path):
    import torch
    ran = []
    monkeypatch.setattr(B, "HERE", str(tmp_path))
    monkeypatch.setattr(B, "OBJ", str(tmp_path))

    def run(cmd):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(B, "_run", run)
    mod = B.build_generation()
    assert os.path.dirname(mod) == str(tmp_path) and len(ran) == 1
    assert B.build_generation() == mod and len(ran) == 1     # nothing has changed
    monkeypatch.setattr(torch, "__version__", "0.0.test")
    B.build_generation()
    assert len(ran) == 2
    B.build_generation()
    assert len(ran) == 2
