"""The library's build does not hang on the binding's, and the binding follows its torch and Python."""

import importlib.util
import warnings

import pytest

from vllm_ascend_hust_latchmoe_b200 import _build, decoder_ops


def test_library_is_built_without_a_host_compiler(monkeypatch, tmp_path):
    """Present sources, no binding and no compiler for it: a warning, and the library all the same."""
    _build.build()
    monkeypatch.setattr(_build, "BINDING_PATH", tmp_path / "_decoder_ops.so")
    monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    with pytest.warns(UserWarning, match="_decoder_ops.so is not built"):
        assert _build.build() == _build.LIB_PATH
    assert not _build.BINDING_PATH.exists()
    with pytest.raises(OSError):
        _build.build_binding()
    # a compiler that fails
    monkeypatch.setenv("CXX", "false")
    with pytest.warns(UserWarning, match="binding's build failed"):
        assert _build.build() == _build.LIB_PATH
    # and the operators say so at their first call
    monkeypatch.setattr(decoder_ops, "BINDING_PATH", _build.BINDING_PATH)
    with pytest.raises(RuntimeError, match="not built"):
        decoder_ops._load()


def test_library_comes_before_the_binding(monkeypatch, tmp_path):
    order = []
    monkeypatch.setattr(_build, "build_library", lambda *a: order.append("library") or _build.LIB_PATH)
    monkeypatch.setattr(_build, "build_binding", lambda *a: order.append("binding"))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert _build.build() == _build.LIB_PATH
    assert order == ["library", "binding"]


def test_binding_of_another_torch_or_python_is_out_of_date(monkeypatch):
    _build.build_binding()
    assert _build.binding_is_current()
    spec = importlib.util.spec_from_file_location("_decoder_ops", _build.BINDING_PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.built_for == _build.binding_key()
    other = _build.binding_key().replace("torch ", "torch 0.")
    monkeypatch.setattr(_build, "binding_key", lambda: other)
    monkeypatch.setattr(decoder_ops, "binding_key", lambda: other)
    assert not _build.binding_is_current()
    with pytest.raises(RuntimeError, match="built for"):
        decoder_ops._load()


def test_failed_rebuild_leaves_no_old_binding(monkeypatch, tmp_path):
    stale = tmp_path / "_decoder_ops.so"
    stale.write_bytes(b"of another torch")
    monkeypatch.setattr(_build, "BINDING_PATH", stale)
    monkeypatch.setenv("CXX", "false")
    with pytest.raises(RuntimeError):
        _build.build_binding()
    assert not stale.exists()
