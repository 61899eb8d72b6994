"""When the torch front-end (_nfx_torch.so) is built, with a stand-in for the compiler."""
import os
import subprocess

import pytest


@pytest.fixture
def front(monkeypatch, tmp_path):
    """(the build module, the list of compiler calls) with outputs under tmp_path."""
    from neuroflow_b200 import build as nb
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(nb, "TORCH_EXT", str(tmp_path / "_nfx_torch.so"))
    monkeypatch.setattr(nb.subprocess, "run", run)
    monkeypatch.setattr(nb, "TORCH_STAMP", str(tmp_path / "stamp"), raising=False)
    return nb, calls


def test_no_torch_no_front_end(front, monkeypatch, capsys):
    """libnfx.so and the command line do not need torch, and neither does their build."""
    import importlib.metadata as md
    nb, calls = front
    version = md.version

    def none(name):
        if name == "torch":
            raise md.PackageNotFoundError(name)
        return version(name)

    monkeypatch.setattr(md, "version", none)
    monkeypatch.setitem(__import__("sys").modules, "torch", None)
    nb._build_torch()
    assert not calls and not os.path.exists(nb.TORCH_EXT)
    assert "torch" in capsys.readouterr().err


def test_another_torch_builds_it_again(front, monkeypatch):
    """The binary is made for one version of torch's C++ interface."""
    import importlib.metadata as md
    nb, calls = front
    version, torch_is = md.version, ["2.11.0"]
    monkeypatch.setattr(md, "version", lambda n: torch_is[0] if n == "torch" else version(n))
    nb._build_torch()
    assert len(calls) == 1
    nb._build_torch()
    assert len(calls) == 1
    torch_is[0] = "2.12.0"
    nb._build_torch()
    assert len(calls) == 2
    nb._build_torch()
    assert len(calls) == 2


def test_ops_without_the_front_end_says_what_to_do(monkeypatch):
    import importlib
    import sys
    import neuroflow_b200
    import neuroflow_b200.ops  # noqa: F401
    monkeypatch.setitem(sys.modules, "neuroflow_b200._nfx_torch", None)
    monkeypatch.delattr(neuroflow_b200, "_nfx_torch", raising=False)
    monkeypatch.delitem(sys.modules, "neuroflow_b200.ops")
    with pytest.raises(ImportError, match="neuroflow_b200.build"):
        importlib.import_module("neuroflow_b200.ops")
