"""Loading a library of another version: refused with what to do about it, whatever it exports."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from ayaka_amd.errors import CapabilityError
from ayaka_amd.hip import _lib

CC = shutil.which("gcc") or shutil.which("cc")


def _load(tmp_path: Path, monkeypatch: pytest.MonkeyPatch, source: str) -> None:
    (tmp_path / "other.c").write_text(source)
    path = tmp_path / "libother.so"
    subprocess.run([CC, "-shared", "-fPIC", "-o", str(path), str(tmp_path / "other.c")], check=True)
    monkeypatch.setattr(_lib, "LIB_PATH", path)
    monkeypatch.setattr(_lib, "_lib", None)
    _lib.lib()


@pytest.mark.skipif(CC is None, reason="no C compiler")
@pytest.mark.parametrize("source,message", [
    # an older library: the version says so before an export of this one is looked for
    ("int ayk_abi_version(void) { return %d; }" % (_lib.ABI_VERSION - 1), "has ABI %d" % (_lib.ABI_VERSION - 1)),
    ("int ayk_abi_version(void) { return %d; }" % _lib.ABI_VERSION, "lacks an export"),
    ("int something_else(void) { return 0; }", "lacks an export"),
])
def test_another_library_is_refused(tmp_path, monkeypatch, source, message) -> None:
    with pytest.raises(CapabilityError, match=message) as refused:
        _load(tmp_path, monkeypatch, source)
    assert "rebuild it" in str(refused.value)
    assert _lib._lib is None


def test_the_built_library_is_of_the_packages_version() -> None:
    # (18 was the version before the block-scaled caches and the step tables)
    assert _lib.lib().ayk_abi_version() == _lib.ABI_VERSION > 18
