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


def test_every_tile_is_written_once_a_wait_ran_out(tmp_path):
    """The pair kernel's results warps, with waits that run out at any of their tiles: each tile is taken once, from
    the failing one on with `ok` false (its results become NaN), and no further wait is made."""
    src, exe = tmp_path / "tiles.cpp", tmp_path / "tiles"
    src.write_text("""
#include "t5e_blocktiles.h"
#include <cstdio>
int main() {
  int wrong = 0;
  for (uint32_t tiles = 0; tiles < 12; ++tiles)
    for (uint32_t step = 1; step < 5; ++step)
      for (uint32_t first = 0; first < step; ++first)
        for (int fail = -1; fail < 12; ++fail) {  // the count-th wait runs out
          int waits = 0, taken[12] = {0}, good[12] = {0};
          uint32_t counts = 0;
          const bool ok = t5e::blockmm::take_tiles(
              first, tiles, step, [&](uint32_t count) { ++waits; return (int)count != fail; },
              [&](uint32_t tile, uint32_t count, bool ok) { ++taken[tile]; good[tile] = ok; wrong += count != counts++; });
          const int mine = tiles > first ? (int)((tiles - first + step - 1) / step) : 0;
          const bool fails = fail >= 0 && fail < mine;
          wrong += ok == fails || waits != (fails ? fail + 1 : mine);
          for (uint32_t t = 0; t < tiles; ++t) {
            const bool my = t >= first && (t - first) % step == 0;
            wrong += taken[t] != (my ? 1 : 0) || good[t] != (my && (!fails || (int)((t - first) / step) < fail));
          }
        }
  std::printf("%d\\n", wrong);
  return wrong != 0;
}
""")
    csrc = nat.LIB_PATH.parents[1] / "csrc"
    subprocess.run(["g++", "-std=c++17", "-I", str(csrc), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.strip() == "0"
