"""The build command's products: what the PyTorch side links against."""

from __future__ import annotations

import re
import subprocess
import sys

import pytest

from tcgen05_b200 import _native as nat
from tcgen05_b200 import build


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


def test_every_result_is_written_once_a_wait_ran_out(tmp_path):
    """The pair kernel's results warps, each with a wait that runs out at another of its tiles: what it had taken by
    then (the failing tile included) and what it spoils behind it are every result once."""
    src, exe = tmp_path / "tiles.cpp", tmp_path / "tiles"
    src.write_text("""
#include "t5e_blocktiles.h"
#include <cstdio>
#include <vector>
template <int BN>
int wrong(uint32_t rows, uint32_t cols, uint32_t clusters, uint32_t seed) {
  const uint32_t p_tiles = (rows + 255) / 256, tiles = p_tiles * ((cols + BN - 1) / BN);
  std::vector<int> seen(rows * cols);
  const auto write = [&](uint32_t row, uint32_t col) { ++seen[row * cols + col]; };
  for (uint32_t cluster = 0; cluster < clusters; ++cluster)
    for (uint32_t warp = 0; warp < 16; ++warp) {  // two blocks of four quarters by two sides
      const uint32_t rank = warp / 8, quarter = warp % 4, side = warp / 4 % 2;
      uint32_t taken = 1 + (seed + warp * 5 + cluster * 3) % 4, tile = cluster;
      for (; taken > 0 && tile < tiles; tile += clusters, --taken)
        for (uint32_t r = 0; r < 32; ++r)
          for (uint32_t c = side * 64; c < BN; c += c % 64 == 63 ? 65 : 1) {
            const uint32_t row = tile % p_tiles * 256 + rank * 128 + quarter * 32 + r, col = tile / p_tiles * BN + c;
            if (row < rows && col < cols) write(row, col);
          }
      for (uint32_t lane = 0; lane < 32; ++lane)
        t5e::blockmm::spoil_tiles<BN>(tile, tiles, clusters, p_tiles, rank * 128 + quarter * 32, side * 64, lane, rows, cols,
                                      write);
    }
  int bad = 0;
  for (int n : seen) bad += n != 1;
  return bad;
}
int main() {
  int bad = 0;
  for (uint32_t seed = 0; seed < 4; ++seed)
    for (uint32_t rows : {1u, 129u, 256u, 700u, 1100u})
      for (uint32_t cols : {1u, 63u, 128u, 300u, 515u, 777u})
        for (uint32_t clusters : {1u, 2u, 5u}) bad += wrong<128>(rows, cols, clusters, seed) + wrong<256>(rows, cols, clusters, seed);
  std::printf("%d\\n", bad);
  return bad != 0;
}
""")
    csrc = nat.LIB_PATH.parents[1] / "csrc"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(csrc), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.strip() == "0"


def test_block_kernels_read_through_ordinary_loads():
    """With programmatic launches a kernel begins while the one before still writes what it will read: no load may be
    of the kind that asks for memory that is read-only all the while, or that a compiler may move ahead of the wait."""
    csrc = nat.LIB_PATH.parents[1] / "csrc"
    for name in ("t5e_blocks.cuh", "t5e_blocks.cu", "t5e_blockmm.cu"):
        code = "\n".join(line.split("//")[0] for line in (csrc / name).read_text().splitlines())
        assert "griddepcontrol.wait" in code or "wait_for_previous_grid" in code
        for word in ("__ldg(", ".nc", "__restrict__", "__ldcg(", "__ldlu("):
            assert word not in code, (name, word)
        assert not re.findall(r"asm\s*\(\s*\"[^;]*\bld\.", code), name


def test_the_c_library_builds_without_pytorch_or_a_cxx_compiler(monkeypatch, capfd):
    monkeypatch.setattr(build, "_build_cuda", lambda *a: build.LIB)
    monkeypatch.setattr(build.subprocess, "run", lambda *a, **k: pytest.fail("a compiler was called"))
    monkeypatch.setenv("CXX", "/nowhere/g++")
    assert build.build(force=True) == build.LIB
    assert "left out: no C++ compiler /nowhere/g++" in capfd.readouterr().err
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build(force=True) == build.LIB
    assert "t5e_torch.so is left out" in capfd.readouterr().err


def test_the_extension_is_rebuilt_for_another_pytorch(monkeypatch):
    import torch

    calls = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **k: calls.append(cmd))
    monkeypatch.setattr(build.os, "replace", lambda a, b: None)
    monkeypatch.setattr(build, "TORCH_SRC", build.INCLUDE / "t5e.h")  # newer sources are not what this is about
    words = f"t5e_torch for torch {torch.__version__} python".encode()
    assert words in build.TORCH_LIB.read_bytes()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    monkeypatch.setenv("CXX", "env g++ -g0")  # a command, not only a path
    build.build_torch()
    assert len(calls) == 1 and calls[0][:3] == ["env", "g++", "-g0"] and any("t5e_torch for torch 0.0.1 python" in str(arg) for arg in calls[0])


def test_an_extension_that_does_not_load_is_named(tmp_path, monkeypatch):
    bad = tmp_path / "t5e_torch.so"
    bad.write_bytes(b"not a library")
    monkeypatch.setattr(nat, "TORCH_LIB_PATH", bad)
    monkeypatch.setattr(nat, "_torch_ops", None)
    with pytest.raises(nat.NativeLibraryError, match="rebuild it"):
        nat.torch_ops()


def test_star_import_without_pytorch():
    """What needs no PyTorch is imported without it; where it is there, the block-scaled calls come along."""
    code = "import sys\n{}\nfrom tcgen05_b200 import *\nprint(make_model('tf32') is not None, 'quantize_blocks' in globals())\n"
    hide = ("import importlib.util as u\nfind = u.find_spec\nu.find_spec = lambda n, *a: None if n == 'torch' else find(n, *a)\n"
            "sys.modules['torch'] = None")
    for first, words in ((hide, "True False"), ("", "True True")):
        r = subprocess.run([sys.executable, "-c", code.format(first)], capture_output=True, text=True,
                           cwd=nat.LIB_PATH.parents[2])
        assert r.stdout.strip() == words, r.stderr[-800:]
