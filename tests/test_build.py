"""The build command's products: what the PyTorch side links against."""

from __future__ import annotations

import subprocess

from tcgen05_b200 import _native as nat


def test_extension_shares_the_cxx_library_of_pytorch():
    """A compiler that links libstdc++ statically (a $CXX of its own) would give an extension whose refusals end the
    process: its streams and libc10's would not know each other's facets."""
    out = subprocess.run(["readelf", "-d", str(nat.TORCH_LIB_PATH)], capture_output=True, text=True, check=True).stdout
    assert "[libstdc++.so.6]" in out
    names = subprocess.run(["nm", "-D", "--defined-only", str(nat.TORCH_LIB_PATH)], capture_output=True, text=True,
                           check=True).stdout
    assert "_ZNSt6locale" not in names
