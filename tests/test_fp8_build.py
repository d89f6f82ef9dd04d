"""Building the 8-bit path's Python module: the library does not need it, and another torch or Python
needs another build (no compiler runs here)."""
import os
import types

import pytest

from flashbfp_b200 import _lib, build, fp8


@pytest.fixture
def place(tmp_path, monkeypatch):
    """A module file of our own, as built for this torch, and the compilations asked for."""
    monkeypatch.setattr(build, "BIND", str(tmp_path / "_fp8_bind.so"))
    monkeypatch.setattr(build, "BIND_STAMP", str(tmp_path / "b" / "stamp"))
    monkeypatch.setattr(build, "_stale", lambda: False)
    runs = []

    def run(cmd, check):
        assert check and cmd[0] == "g++"
        runs.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("module")

    monkeypatch.setattr(build.subprocess, "run", run)
    return runs


@pytest.mark.parametrize("lacks", ["torch", "g++", "Python.h"])
def test_the_library_builds_without_what_only_the_module_needs(place, monkeypatch, capsys, tmp_path, lacks):
    if lacks == "torch":
        find = build.importlib.util.find_spec
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None if name == "torch" else find(name))
    elif lacks == "g++":
        monkeypatch.setattr(build.shutil, "which", lambda name: None)
    else:
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert build.build() == build.LIB
    assert not place and not os.path.exists(build.BIND)
    assert lacks in capsys.readouterr().err
    monkeypatch.setattr(fp8, "_bind", None)
    monkeypatch.setattr(_lib, "lib", lambda: None)
    with pytest.raises(_lib.FlashBFPError, match="missing"):
        fp8._module()


def test_another_torch_builds_again(place, monkeypatch, capsys):
    build.build()
    assert len(place) == 1 and os.path.exists(build.BIND)
    build.build()
    assert len(place) == 1                               # up to date
    monkeypatch.setattr(build, "bind_for", lambda: "torch 9.9, Python 3.99")
    build.build()
    assert len(place) == 2
    assert any("torch 9.9, Python 3.99" in a for a in place[1])
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    build.build()                                        # nothing to do: no compiler needed, no note
    assert len(place) == 2 and not capsys.readouterr().err


def test_a_module_of_unknown_origin_is_built_again(place):
    build.build()
    os.remove(build.BIND_STAMP)
    build.build()
    assert len(place) == 2


def test_a_module_for_another_torch_is_refused(place, monkeypatch):
    build.build()
    monkeypatch.setattr(fp8, "_bind", None)
    monkeypatch.setattr(_lib, "lib", lambda: None)
    module = types.SimpleNamespace(built_for="torch 1.0, Python 3.8", setup=lambda *a: pytest.fail("used"))
    loader = types.SimpleNamespace(exec_module=lambda m: None)
    monkeypatch.setattr(fp8.importlib.util, "spec_from_file_location",
                        lambda name, path: types.SimpleNamespace(loader=loader))
    monkeypatch.setattr(fp8.importlib.util, "module_from_spec", lambda spec: module)
    with pytest.raises(_lib.FlashBFPError, match="built for torch 1.0, Python 3.8"):
        fp8._module()
    assert fp8._bind is None


def test_the_built_module_is_for_this_torch():
    build.build()
    assert fp8._module().built_for == build.bind_for()
