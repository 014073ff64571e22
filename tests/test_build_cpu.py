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


def test_entry_points_carry_their_interpreters_tag():
    """One Python version does not load what another's headers built."""
    import sysconfig
    assert os.path.basename(B.FASTCALL) == "_fastcall" + sysconfig.get_config_var("EXT_SUFFIX")
    from clove_compute_b200 import _lib
    assert os.path.samefile(_lib.fastcall().__file__, B.FASTCALL)


def test_untagged_entry_points_are_removed(monkeypatch, tmp_path):
    """A file of the old name, which every version would load, goes with the next build."""
    old = tmp_path / "_fastcall.so"
    old.write_bytes(b"old")
    monkeypatch.setattr(B, "FASTCALL", str(tmp_path / ("_fastcall" + B.sysconfig.get_config_var("EXT_SUFFIX"))))
    B._build_fastcall(False)
    assert not old.exists() and os.path.exists(B.FASTCALL)
