"""The decode binding's file belongs to one Python and one PyTorch (no GPU)."""
import pytest
import torch

from tread_b200 import _capi, build


def test_another_pytorch_has_another_file(monkeypatch):
    here = _capi.binding_path()
    assert torch.__version__ in here
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert _capi.binding_path() != here
    monkeypatch.setattr(_capi, "_binding", None)
    with pytest.raises(RuntimeError, match="not built for this Python and PyTorch.*python -m tread_b200.build"):
        _capi.binding()


def test_a_build_for_another_pytorch_is_stale(monkeypatch, tmp_path):
    """build() compiles the binding again, and takes away the file of the other version."""
    for name in ("OUT_DIR", "OBJ_DIR"):
        monkeypatch.setattr(build, name, str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libtread_b200.so"))
    monkeypatch.setattr(_capi, "LIB_PATH", str(tmp_path / "libtread_b200.so"))
    compiled = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, check: compiled.append(cmd[cmd.index("-o") + 1]))
    old, other = tmp_path / "tread_decode.cpython-1-torch1.so", tmp_path / "tread_decode.so"
    old.write_bytes(b""), other.write_bytes(b"")
    build.build()
    assert compiled[-1] == _capi.binding_path() and not old.exists() and not other.exists()
    open(_capi.binding_path(), "w").close()
    compiled.clear()
    build.build()
    assert _capi.binding_path() not in compiled
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build()
    assert compiled[-1] == _capi.binding_path()
