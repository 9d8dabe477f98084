"""The native build where torch is absent or was changed: the library with the C ABI needs none of it."""
import importlib.metadata
import sys

import pytest

from megcc_b200 import build


@pytest.fixture
def steps(monkeypatch, tmp_path):
    """Compilers that only note what they were to make."""
    made = []

    class Done:
        returncode, stdout = 0, ""

        def __init__(self, cmd, **_):
            target = cmd[cmd.index("-o") + 1]
            made.append(target)
            with open(target, "wb") as f:
                f.write(" ".join(cmd).replace('"', "\0").encode())

        def communicate(self):
            return "", None

    monkeypatch.setattr(build.subprocess, "run", Done)
    monkeypatch.setattr(build.subprocess, "Popen", Done)
    monkeypatch.setattr(build, "TORCHCALL", str(tmp_path / "_torchcall.so"))
    return made


def test_without_torch_all_else_is_built(steps, monkeypatch, tmp_path, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    monkeypatch.setattr(build, "LIB", str(tmp_path / "library.so"))
    monkeypatch.setattr(build, "_stale", lambda target, deps: target.startswith(str(tmp_path)))
    assert build.build() == str(tmp_path / "library.so")
    assert steps == [str(tmp_path / "library.so")]
    assert "_torchcall.so" in capsys.readouterr().err


def test_another_torch_makes_the_module_anew(steps, monkeypatch):
    assert build.build_torchcall() == build.TORCHCALL and len(steps) == 1
    assert build.build_torchcall() == build.TORCHCALL and len(steps) == 1  # (nothing changed)
    real = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "99.0" if name == "torch" else real(name))
    assert build.build_torchcall() == build.TORCHCALL and len(steps) == 2


def test_the_library_comes_first(steps, monkeypatch, tmp_path):
    order = []
    monkeypatch.setattr(build, "build_torchcall", lambda *a: order.append("calls") or 1 / 0)
    monkeypatch.setattr(build, "LIB", str(tmp_path / "library.so"))
    monkeypatch.setattr(build, "_stale", lambda target, deps: target.startswith(str(tmp_path)))
    with pytest.raises(ZeroDivisionError):
        build.build()
    assert steps == [str(tmp_path / "library.so")]
