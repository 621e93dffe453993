"""What build.build() compiles when the torch side of the training operators cannot be."""
import subprocess
import types

import pytest

from puffysics_b200 import build


@pytest.fixture
def commands(monkeypatch):
    """The commands that build.build() runs, none of them for real: all but torch's side and the step library is up to date."""
    got = []

    def run(cmd, **_):
        got.append(cmd)
        return types.SimpleNamespace(returncode=int(build.TRAIN_PY_SRC in cmd), stdout="", stderr="no such header")
    monkeypatch.setattr(build, "subprocess", types.SimpleNamespace(run=run, Popen=subprocess.Popen, PIPE=subprocess.PIPE,
                                                                   STDOUT=subprocess.STDOUT))
    monkeypatch.setattr(build, "_newer", lambda out, deps: out in (build.LIB, build.TRAIN_PY_LIB))
    return got


def has(commands, lib):
    return any(lib in cmd for cmd in commands)


def test_the_step_library_builds_without_torch(commands, monkeypatch, capsys):
    find = build.importlib.util.find_spec
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build() == build.LIB
    assert has(commands, build.LIB) and not has(commands, build.TRAIN_PY_LIB)
    assert "torch" in capsys.readouterr().err
    monkeypatch.setattr(build, "_newer", lambda out, deps: out == build.TRAIN_PY_LIB)
    assert build.up_to_date()


def test_the_step_library_builds_beside_a_torch_that_does_not_compile(commands):
    with pytest.raises(RuntimeError, match="no such header"):
        build.build()
    assert has(commands, build.LIB) and has(commands, build.TRAIN_PY_LIB)


def test_the_torch_side_follows_the_installed_torch(monkeypatch):
    """A library built against another torch's headers is stale for the build, and not loaded."""
    from puffysics_b200 import train
    build.build()
    assert build.train_py_up_to_date() and train._binding()
    assert build.torch_version() in build.built_for()
    monkeypatch.setattr(build, "torch_version", lambda: "99.0")
    assert not build.train_py_up_to_date() and not build.up_to_date()
    monkeypatch.setattr(train, "_py", None)
    with pytest.raises(RuntimeError, match="99.0"):
        train._binding()
