"""Where the attention kernels read and write: their index arithmetic
(attend_index.h), compiled for the host and run for every workgroup."""

import ctypes
import subprocess

import numpy as np
import pytest

from nkipy_amd import _build
from nkipy_amd.dispatch import serving as S

HARNESS = r"""
#include <algorithm>
#include <vector>
#define NK_DEVICE inline
using std::max;
using std::min;
template <typename F> static int att_find(int n, int x, F f) {  // as the wave counts
  int c = 0;
  for (int b = 0; b < n; ++b) c += f(b) <= x;
  return c - 1;
}
#include "attend_index.h"
using namespace nk;

// rows read or written outside the tensors; how often each (query, head) is written
extern "C" int64_t tiles(const AttendArgs *args, int32_t *written) {
  const AttendArgs &a = *args;
  const int rep = a.Hq / a.Hkv;
  int64_t outside = 0;
  for (int w = 0; w < a.tiles * a.Hkv * a.nsplit; ++w) {
    AttWork k;
    AttSeq s;
    if (!att_tile<true>(a, w, k, s)) continue;
    const AttSpan sp = att_span(a, s, k.tile);
    int j0, j1;
    if (k.split >= att_split(a, sp.nb, k.split, j0, j1)) continue;
    if (k.b >= a.B || k.g >= a.Hkv) ++outside;
    const int rows = s.n * rep;
    for (int l = 0; l < ATT_ROWS; ++l) {
      const int row = k.tile * ATT_ROWS + l, rld = min(row, rows - 1), t = s.lo + rld / rep, h = k.g * rep + rld % rep;
      if (t < 0 || t >= a.N || h < 0 || h >= a.Hq) ++outside;
      else if (row < rows && k.split == 0) ++written[(int64_t)t * a.Hq + h];
    }
    for (int j = j0; j < j1; ++j)
      for (int x = 0; x < ATT_KEYS; ++x) {
        const int key = sp.kb(j) * ATT_KEYS + x;
        if (key >= sp.hi || (key < sp.lo && key >= a.sinks)) continue;
        if (key < 0 || key / a.page >= a.width) ++outside;
        else if (att_place(a, k.b, key) >= a.pages * a.pitch) ++outside;
      }
  }
  // row by row, as the form without tiles and the joining launch look for them
  for (int t = 0; t < a.N; ++t) {
    int b, i;
    AttSeq s;
    if (att_query(a, t, b, s, i) && (b >= a.B || i < 0 || i >= s.n || s.lo + i != t)) ++outside;
  }
  return outside;
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("index")
    (d / "index.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", f"-I{_build.KERNEL_DIR}", str(d / "index.cpp"), "-o",
                    str(d / "index.so")], check=True)
    lib = ctypes.CDLL(str(d / "index.so"))
    lib.tiles.restype = ctypes.c_int64
    return lib


def tiles(index, starts, lens, n, hq, hkv, page=16, width=8, pages=20, window=0, sinks=0):
    """(accesses outside the tensors, how often each row is written) of the tiled form."""
    starts, lens = np.array(starts, np.int64).astype(np.int32), np.array(lens, np.int64).astype(np.int32)
    tables = np.random.default_rng(0).integers(-2, pages + 2, (len(lens), width)).astype(np.int32)
    a = S.AttendArgs()
    S._fields(a, tables=tables.ctypes.data, lens=lens.ctypes.data, starts=starts.ctypes.data, B=len(lens), S=1, N=n, Hq=hq,
              Hkv=hkv, D=64, page=page, pages=pages, width=width, pitch=page, window=window or S.NO_WINDOW, sinks=sinks,
              min_blocks=S.ATT_TILE_BLOCKS)
    _, a.tiles, a.nsplit = S.attend_work(len(lens), 1, n, hq, hkv, 64, width * page, window, sinks, True)
    written = np.zeros((n, hq), np.int32)
    return index.tiles(ctypes.byref(a), ctypes.c_void_p(written.ctypes.data)), written


@pytest.mark.parametrize("hq,hkv", [(8, 4), (4, 1), (3, 3), (17, 1), (256, 1)])
def test_tiles_cover_each_row_once(index, hq, hkv):
    rng = np.random.default_rng(1)
    for _ in range(30):
        new = rng.integers(0, rng.choice([2, 40, 300]), rng.integers(1, 70))
        starts = np.concatenate([[0], np.cumsum(new)]) + rng.integers(0, 9)
        n = int(starts[-1]) + int(rng.integers(1, 9))
        outside, written = tiles(index, starts, new + rng.integers(0, 100, len(new)), n, hq, hkv, window=int(rng.choice([0, 40])))
        assert outside == 0
        assert (written[starts[0]:starts[-1]] == 1).all() and written.sum() == (starts[-1] - starts[0]) * hq


@pytest.mark.parametrize("hq,hkv", [(8, 4), (4, 1), (3, 3), (17, 1), (256, 1)])
def test_tiles_of_unordered_starts_stay_inside(index, hq, hkv):
    """Starts and lengths that make no sense, of batches long enough that a sequence's
    first tile lies behind tiles that look for it."""
    rng = np.random.default_rng(2)
    far = [2**31 - 1, -2**31]
    for starts in ([0, 1000, 0, 1000], [1000, 0, 0, 0], [700, 3, 900, 900], far * 2, [0] + far + [1000]):
        for lens in ([100, 100, 100], [2**31 - 1, -2**31, 7]):
            assert tiles(index, starts, lens, 1000, hq, hkv)[0] == 0
    for _ in range(60):
        b = int(rng.integers(1, 40))
        n = int(rng.integers(1, 2000))
        starts = rng.integers(-n, 2 * n + 1, b + 1)
        lens = rng.integers(-10, 400, b)
        assert tiles(index, starts, lens, n, hq, hkv, window=int(rng.choice([0, 20])), sinks=1)[0] == 0
