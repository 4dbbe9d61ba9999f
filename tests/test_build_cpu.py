"""The build of the Python call path (zealot_b200/build.py) on machines that lack what it needs."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(ROOT, "zealot_b200", "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    monkeypatch.setattr(m, "CALLS", str(tmp_path / "calls.so"))
    return m


def test_without_torch_the_library_alone_is_built(build, monkeypatch, capsys):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    assert os.path.exists(build.build())
    assert not os.path.exists(build.CALLS) and "torch" in capsys.readouterr().err


def test_without_python_headers_the_library_alone_is_built(build, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert os.path.exists(build.build())
    assert not os.path.exists(build.CALLS) and "Python.h" in capsys.readouterr().err


def test_a_call_path_that_does_not_compile_is_an_error(build, monkeypatch):
    monkeypatch.setattr(build, "INCLUDE", os.path.join(ROOT, "zealot_b200"))  # no zealot_attn.h there
    monkeypatch.setattr(build.os.path, "getmtime", lambda path: 0)
    with pytest.raises(RuntimeError, match="gcc failed"):
        build._build_calls(force=True)


def test_the_call_path_is_built_where_both_are(build):
    build._build_calls(force=False)
    assert os.path.exists(build.CALLS)
