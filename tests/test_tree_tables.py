"""The tables that the attention of new rows reads, checked entry by entry: its functions that cut the work
are compiled for the CPU as they stand in the source, with every table behind a pointer that knows its
length.  (On the GPU a value read behind a table is thrown away, so no result shows it.)"""
import ctypes
import pathlib
import re
import shutil
import subprocess

import pytest

from yirage_amd import _lib
from yirage_amd._lib import lib

CSRC = pathlib.Path(_lib.__file__).parent / "csrc"

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")

HEAD = r"""
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#define __device__
#define __forceinline__ inline
#define YR_G
using std::max; using std::min;
struct int4 { int x, y, z, w; };
static struct { int x; } threadIdx;
constexpr int kWave = 64;
// the tables: [address, entries]; a read outside of its own is counted
struct Table { const int32_t* p; long n; };
static Table tables[4];
static long outside = 0;
struct Checked {
  const int32_t* p;
  int32_t operator[](long i) const {
    for (const Table& t : tables)
      if (t.p == p) { if (i < 0 || i >= t.n) { outside++; return 0; } return p[i]; }
    abort();
  }
};
static Checked gptr(const int32_t* p) { return Checked{p}; }
// what lanes do together: not part of what is compiled here
static long long scan64(long long) { abort(); }
static long long lane64(long long, int) { abort(); }
static uint64_t __ballot(bool) { abort(); }
static int __builtin_amdgcn_readlane(int, int) { abort(); }
"""
TAIL = r"""
}
using namespace yr;
// every workgroup of a call without qo_indptr, `parts` of a kv head, whose tokens are not split ->
// reads outside of the tables, workgroups that found a sequence
extern "C" void walk(int batch, int parts, int tt, long* result2) {
  int32_t* len = new int32_t[batch]; int32_t* ptr = new int32_t[batch + 1]; int32_t ids = 0;
  for (int b = 0; b < batch; b++) len[b] = 100;
  for (int b = 0; b <= batch; b++) ptr[b] = 0;
  tables[0] = {len, batch}; tables[1] = {ptr, batch + 1}; tables[2] = {&ids, 1};
  TreeArgs a = {};
  a.r = Ragged{nullptr, ptr, &ids, len, batch, batch, 16, 1, 1};
  a.tt = tt;
  a.parts = parts;
  outside = 0;
  result2[1] = 0;
  for (int lane = 0; lane < kWave; lane++) seq_work(a, lane);
  for (int w = 0; w < parts; w++) {
    const TileAt t = find_index(a, SeqWork{}, w);
    if (t.b < batch) result2[1]++;
  }
  result2[0] = outside;
  delete[] len; delete[] ptr;
}
"""


def _cut(text, start, end="\n}"):
    """The definition that begins with `start`, to its closing brace at the line's front."""
    at = text.index(start)
    stop = text.index(end, at) + len(end)
    return text[at:stop] + (";" if text[stop:stop + 1] == ";" else "") + "\n"


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("tables")
    ragged = re.sub(r'#pragma once|#include "yr_common.h"', "", (CSRC / "ragged.h").read_text())
    tree = (CSRC / "tree_attn.hip").read_text()
    parts = [re.search(r"constexpr int TR_TILE_COST = \d+;", tree)[0] + "\n"]
    parts += [_cut(tree, s) for s in ("struct TreeArgs {", "struct SeqWork {", "__device__ __forceinline__ long long units_before(",
                                      "__device__ __forceinline__ SeqWork seq_work(", "struct TileAt {",
                                      "__device__ __forceinline__ SeqRows seq_of_lane(", "__device__ __forceinline__ TileAt find_index(")]
    (d / "walk.cc").write_text(HEAD + ragged + "namespace yr {\n" + "".join(parts) + TAIL)
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-shared", "-fPIC", "-o", "walk.so", "walk.cc"], cwd=d, check=True)
    return ctypes.CDLL(str(d / "walk.so")).walk


@pytest.mark.parametrize("hkv", [1, 2, 8])
@pytest.mark.parametrize("batch", [1, 2, 31, 40])
@pytest.mark.parametrize("most", [0, 600, 4096])
def test_single_rows_read_their_own_tables(walk, batch, hkv, most):
    """Single rows without qo_indptr, in a call made for tokens to split that turn out to be few."""
    plan, result = (ctypes.c_int * 3)(), (ctypes.c_long * 2)()
    assert lib().yr_hip_gqa_tree_plan(batch, batch, 0, 4 * hkv, hkv, 128, most, _lib.DTYPE_BF16, plan) == 0
    assert plan[2] > 0  # (workgroups of a kv head)
    walk(batch, plan[2], plan[1], result)
    assert result[0] == 0, "reads behind kv_len or kv_indptr"
    assert result[1] == min(batch, plan[2])
