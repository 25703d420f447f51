"""The build command's products: what the PyTorch side links against."""

from __future__ import annotations

import subprocess

import pytest

from tcgen05_b200 import _native as nat


def test_extension_shares_the_cxx_library_of_pytorch():
    """A compiler that links libstdc++ statically (a $CXX of its own) would give an extension whose refusals end the
    process: its streams and libc10's would not know each other's facets."""
    out = subprocess.run(["readelf", "-d", str(nat.TORCH_LIB_PATH)], capture_output=True, text=True, check=True).stdout
    assert "[libstdc++.so.6]" in out
    names = subprocess.run(["nm", "-D", "--defined-only", str(nat.TORCH_LIB_PATH)], capture_output=True, text=True,
                           check=True).stdout
    assert "_ZNSt6locale" not in names


@pytest.mark.parametrize("source,words", [("int t5e_abi_version(void) { return 1; }", "ABI version 1, expected .*rebuild"),
                                          ("int other;", "not the emulator library")])
def test_a_library_of_another_version_is_named(tmp_path, monkeypatch, source, words):
    """An older library lacks functions that this package binds; the message is the version's, not a missing name."""
    src, lib = tmp_path / "old.c", tmp_path / "libt5e.so"
    src.write_text(source + "\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(lib)], check=True)
    monkeypatch.setattr(nat, "LIB_PATH", lib)
    monkeypatch.setattr(nat, "_lib", None)
    with pytest.raises(nat.NativeLibraryError, match=words):
        nat.load()
