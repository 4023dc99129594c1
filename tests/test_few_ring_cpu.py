"""The few-token kernels' rings on the host: which slots are on their way whenever a wait gives up."""

from __future__ import annotations

import ctypes as C
import shutil
import subprocess

import pytest

from conftest import PKG

SOURCE = r"""
#include "few_ring.cuh"

// Chunks through a ring as the kernels take them: all slots filled, then one taken and (as long
// as there are chunks) filled again, with the refill `late` chunks behind.  Before every take:
// the fillings that have not been taken are those that ahead() gives first, in their order, each
// with its own phase.  Returns the first chunk at which that fails, or -1.
extern "C" int run(int depth, int chunks, int late) {
  sb::FewSlots ring(depth);
  int filled[16] = {}, taken[16] = {}, next = 0, used[16];
  auto fill = [&](int slot) {
    if (next == chunks) return;
    ++next;
    ++filled[slot];
  };
  for (int d = 0; d < depth; ++d) fill(d);
  int waiting = 0;
  for (int c = 0; c < chunks; ++c) {
    const int flying = next - c;
    if (flying < 1 || flying > depth) return c;
    for (int i = 0; i < depth; ++i) {
      uint32_t phase;
      const int slot = ring.ahead(i, &phase);
      if (slot != (c + i) % depth || filled[slot] != taken[slot] + (i < flying)) return c;
      if (phase != (uint32_t)(taken[slot] & 1)) return c;
    }
    const int slot = ring.out;
    ring.taken();
    if (slot != c % depth) return c;
    ++taken[slot];
    used[waiting++] = slot;
    if (waiting > late) {
      fill(used[0]);
      for (int i = 1; i < waiting; ++i) used[i - 1] = used[i];
      --waiting;
    }
  }
  return next == chunks ? -1 : chunks;
}
"""


def test_slots_on_their_way(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    (tmp_path / "ring.cpp").write_text(SOURCE)
    so = tmp_path / "ring.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(PKG / "csrc"), "-o", str(so),
                    str(tmp_path / "ring.cpp")], check=True)
    run = C.CDLL(str(so)).run
    for depth in range(2, 9):
        for chunks in (1, 2, depth - 1, depth, depth + 1, 5 * depth + 3):
            for late in (0, 1):
                assert run(depth, chunks, late) == -1, (depth, chunks, late)


def test_every_ring_waits_in_one_place():
    """A wait that runs out there goes on to the copies on their way, slot by slot."""
    text = "".join((PKG / "csrc" / name).read_text() for name in ("few_stream.cuh", "moe_few.cu"))
    assert text.count("mbar_wait_warp(") == 1 == text.count("lost = !few_ring_wait(")
    assert "i < slots.depth" in text and "slots.ahead(i, &phase)" in text
