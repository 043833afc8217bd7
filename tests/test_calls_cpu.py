"""The small extension for the decode step's calls belongs to one interpreter, and nobody depends on it."""
import importlib
import importlib.util
import shutil
import sysconfig
from pathlib import Path

import pytest

import __graft_entry__ as ge

SUFFIX = sysconfig.get_config_var("EXT_SUFFIX")


@pytest.fixture
def capi(pkg):
    module = importlib.import_module(pkg.__name__ + ".capi")
    kept, module._CALLS = module._CALLS, None
    yield module
    module._CALLS = kept


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py with its folders in tmp_path."""
    spec = importlib.util.spec_from_file_location("_w8a8_build_test", ge.PKG_DIR / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    if not Path(sysconfig.get_paths()["include"], "Python.h").exists() or not shutil.which("g++"):
        pytest.skip("no Python headers or no g++")
    (tmp_path / "csrc").mkdir()
    (tmp_path / "lib").mkdir()
    monkeypatch.setattr(b, "CSRC", tmp_path / "csrc")
    monkeypatch.setattr(b, "LIB", tmp_path / "lib" / "libw8a8.so")
    return b


def test_the_extension_carries_the_interpreters_suffix(capi, builder, tmp_path, monkeypatch):
    assert SUFFIX != ".so"
    shutil.copy(ge.PKG_DIR / "csrc" / "w8a8_calls.cpp", builder.CSRC)
    made = builder.build_calls()
    assert made == tmp_path / "lib" / ("w8a8_calls" + SUFFIX) and made.exists()
    assert capi._calls_path().name == made.name
    monkeypatch.setattr(capi, "_calls_path", lambda: made)
    assert not isinstance(capi._load_calls(capi.load_library()), capi._CtypesCalls)


def test_another_interpreters_extension_is_not_looked_at(capi, tmp_path, monkeypatch):
    for name in ("w8a8_calls.so", "w8a8_calls.cpython-27-none.so"):
        (tmp_path / name).write_bytes(b"not for this one")
    path = capi._calls_path()
    monkeypatch.setattr(capi, "_calls_path", lambda: tmp_path / path.name)
    assert isinstance(capi._load_calls(capi.load_library()), capi._CtypesCalls)


def test_an_extension_that_does_not_load_is_done_without(capi, tmp_path, monkeypatch):
    broken = tmp_path / ("w8a8_calls" + SUFFIX)
    broken.write_bytes(b"no shared object")
    monkeypatch.setattr(capi, "_calls_path", lambda: broken)
    with pytest.warns(RuntimeWarning, match="ctypes"):
        calls = capi._load_calls(capi.load_library())
    assert isinstance(calls, capi._CtypesCalls)
    assert calls.w8a8_unpack_weight4(None, None, 2, 2, None, None) != 0  # (refused: no context)


def test_a_failing_compiler_leaves_no_extension_behind(builder, capsys):
    (builder.CSRC / "w8a8_calls.cpp").write_text("no such thing as this;\n")
    old = builder.LIB.parent / ("w8a8_calls" + SUFFIX)
    old.write_bytes(b"of an older source")
    assert builder.build_calls(force=True) is None
    assert not old.exists() and "ctypes" in capsys.readouterr().err
