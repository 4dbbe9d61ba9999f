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
    monkeypatch.setattr(m, "_sources", lambda: [])  # the library that is there, not compiled again
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


def _python(code):
    import subprocess
    import sys
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)


def test_the_package_without_its_call_path():
    """Only the calls that go through it are refused, in words; what does not need it works."""
    r = _python("""
import sys
sys.modules["zealot_b200.calls"] = None  # importing it fails
import torch
import zealot_b200 as zb
assert zb.BlockManager(4, 16).allocate().block_id >= 0
class Context:
    device, lib, address = 0, zb.lib, 0
x = torch.zeros((1, 1, 4))
try:
    zb.CudaAttention(Context()).select_blocks(x, x, x, 16)
except ImportError as e:
    assert "build.py" in str(e), e
else:
    assert False
""")
    assert r.returncode == 0, r.stderr


def test_the_call_path_is_one_for_each_python(build):
    import sysconfig
    from zealot_b200 import calls
    assert os.path.basename(calls.__file__) == "calls" + sysconfig.get_config_var("EXT_SUFFIX")
    assert not os.path.exists(os.path.join(os.path.dirname(calls.__file__), "calls.so"))
