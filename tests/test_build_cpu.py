"""The build on machines that lack what only the paged operators' CPython entry points need."""
import os

import pytest

from clove_compute_b200 import build as B


@pytest.mark.parametrize("lacks", ["headers", "compiler"])
def test_library_is_built_without_the_python_entry_points(monkeypatch, tmp_path, capsys, lacks):
    """Without Python's headers or a C compiler the library itself is still delivered; the
    entry points are left out, with a message, and an outdated file of theirs goes."""
    out = tmp_path / "_fastcall.so"
    out.write_bytes(b"outdated")
    os.utime(out, (1, 1))
    monkeypatch.setattr(B, "FASTCALL", str(out))
    if lacks == "headers":
        monkeypatch.setattr(B.sysconfig, "get_path", lambda name: str(tmp_path))
    else:
        monkeypatch.setattr(B.shutil, "which", lambda name: None)
    B._build_fastcall(False)
    assert not out.exists()
    assert "paged" in capsys.readouterr().err
