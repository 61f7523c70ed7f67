"""A library or an extension built from older sources is refused with the command that rebuilds it. No GPU needed."""
import subprocess
import types

import pytest

from dooms_amd import _lib
from dooms_amd import attention as A


def test_library_without_an_entry_point(monkeypatch, tmp_path):
    src = tmp_path / "old.c"
    src.write_text("\n".join(f"int {f}(void) {{ return 3; }}" for f in _lib.EXPORTS if "paged" not in f))
    old = tmp_path / "libold.so"
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(old)], check=True)
    monkeypatch.setattr(_lib, "LIB_PATH", str(old))
    monkeypatch.setattr(_lib, "_lib", None)
    with pytest.raises(ImportError, match="mx_paged_store.*dooms_amd.build"):
        _lib.lib()
    assert _lib._lib is None


def test_extension_without_the_paged_calls(monkeypatch):
    old = types.SimpleNamespace(bind=lambda *a: None)
    monkeypatch.setattr(A, "_bound", None)
    monkeypatch.setattr(A, "_ext", None)
    monkeypatch.setattr(A.importlib, "import_module", lambda *a: old)
    with pytest.raises(ImportError, match="dooms_amd.build"):
        A._native()
    assert A._bound is None
