"""When build() makes the module through which Python calls the decode-step operators."""
import os
import subprocess

import pytest

import clove_compute_amd.build as b


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    """_build_binding in a folder of its own, with a compiler that only counts."""
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(b, "OBJ", str(tmp_path))
    monkeypatch.setattr(b, "BINDING", str(tmp_path / "_decode.so"))
    monkeypatch.setattr(b.subprocess, "run", run)
    return calls


def test_without_torch_the_module_is_left_out(compiled, monkeypatch, capsys):
    monkeypatch.setattr(b.importlib.util, "find_spec", lambda name: None)
    b._build_binding(True)
    assert not compiled and not os.path.exists(b.BINDING) and "no torch" in capsys.readouterr().err


def test_built_again_for_another_python_or_torch(compiled, monkeypatch):
    pytest.importorskip("torch")
    b._build_binding(False)
    b._build_binding(False)
    assert len(compiled) == 1
    version = b.importlib.metadata.version
    monkeypatch.setattr(b.importlib.metadata, "version", lambda name: version(name) + "+other")
    b._build_binding(False)
    assert len(compiled) == 2
    tag = b.sysconfig.get_config_var
    monkeypatch.setattr(b.sysconfig, "get_config_var", lambda name: "cpython-999" if name == "SOABI" else tag(name))
    b._build_binding(False)
    b._build_binding(False)
    assert len(compiled) == 3
