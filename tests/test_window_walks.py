"""The records by which the windowed attention's backward joins the walks that it cut
between CTAs (csrc/window.cuh), on the CPU: a walk whose records are whole finds all of
its shares, and one whose records were never written ends inside the array."""

import ctypes as C
import shutil
import subprocess

import numpy as np
import pytest

from conftest import PKG_ROOT, REPO

SRC = """
#include "window.cuh"
extern "C" int walk(const int4* pieces, int slots, int slot, int* visited) {
  int steps = pieces[slot].z, n = 0;
  for (int s = slot; s >= 0; s = kda::next_share(pieces, slots, s, pieces[slot].w, &steps)) {
    if (n == slots) return -1;  // goes round and round
    visited[n++] = s;
  }
  return n;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    d = tmp_path_factory.mktemp("walks")
    (d / "walk.cu").write_text(SRC)
    r = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
                        "-I", str(PKG_ROOT / "csrc"), "-I", str(REPO / "include"), str(d / "walk.cu"), "-o",
                        str(d / "walk.so")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    fn = C.CDLL(str(d / "walk.so")).walk

    def visit(pieces, slot):
        assert pieces.dtype == np.int32 and pieces.flags.c_contiguous
        seen = np.full(len(pieces), -1, np.int32)
        n = fn(pieces.ctypes.data_as(C.c_void_p), len(pieces), slot, seen.ctypes.data_as(C.c_void_p))
        assert n >= 0
        return seen[:n].tolist()
    return visit


def records(rng, ctas):
    """Walks of random lengths, cut where equal runs of them end: the records, and the slots
    of each cut walk's shares."""
    lengths = rng.integers(1, 60, size=rng.integers(1, 40))
    ctas = min(ctas, int(lengths.sum()))
    total, start = int(lengths.sum()), np.concatenate([[0], np.cumsum(lengths)])
    pieces, shares = np.zeros((2 * ctas, 4), np.int32), {}
    for c in range(ctas):
        x, end = total * c // ctas, total * (c + 1) // ctas
        while x < end:
            j = int(np.searchsorted(start, x, side="right")) - 1
            it0, walk = x - int(start[j]), int(lengths[j])
            n = min(end - x, walk - it0)
            if n < walk:
                slot = 2 * c + (1 if it0 == 0 else 0)
                pieces[slot] = (0, j, n, walk)
                shares.setdefault(j, []).append(slot)
            x += n
    return pieces, shares


def test_whole_records_give_all_shares(walk):
    rng = np.random.default_rng(0)
    cut = 0
    for _ in range(300):
        pieces, shares = records(rng, int(rng.integers(1, 30)))
        for slots in shares.values():
            assert slots[0] % 2 == 1 and walk(pieces, slots[0]) == slots
            cut += len(slots) > 2
    assert cut > 100


@pytest.mark.parametrize("n", [0, -1, 1, -2 ** 31, 2 ** 31 - 1])
def test_missing_or_stale_records_end_inside_the_array(walk, n):
    rng = np.random.default_rng(1)
    for _ in range(300):
        pieces, shares = records(rng, int(rng.integers(1, 30)))
        lost = rng.random(len(pieces)) < 0.5
        lost[[s[0] for s in shares.values()]] = False  # the join starts at these
        pieces[lost] = rng.integers(-5, 5, size=4)
        pieces[lost, 2] = n
        for slots in shares.values():
            seen = walk(pieces, slots[0])
            assert seen == sorted(set(seen)) and seen[0] == slots[0] and seen[-1] < len(pieces)


def test_a_walk_that_never_gets_its_steps_ends_at_the_last_record(walk):
    pieces = np.zeros((12, 4), np.int32)
    pieces[:] = (0, 0, 1, 1000)
    assert walk(pieces, 1) == [1, 2, 4, 6, 8, 10] and walk(pieces, 11) == [11]
