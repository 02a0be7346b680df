// What the operators on a ragged batch over a paged cache share.
#pragma once
#include "yr_common.h"

namespace yr {

// Sequence b of `batch` owns the rows qo_indptr[b] .. qo_indptr[b + 1) of the
// new tokens (qo_indptr null: row b alone), the pages kv_indices[kv_indptr[b] ..
// kv_indptr[b + 1]) and kv_len[b] tokens, the new ones last.  These tables are
// device data that no host check sees: everything read from them is clamped to
// the sizes the host knows (rows, n_indices, num_pages) before it is used.
// More tokens than one head's keys and values leave room for; with pages of at
// most kMaxPage tokens no position or page end leaves 32 bits.
constexpr int kMaxTokens = 1 << 30, kMaxPage = 1 << 20;

struct Ragged {
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_len;
  int rows, batch, page, n_indices, num_pages;
};

struct SeqRows {
  int row0, n, len;  // first row, rows, tokens
  int pg0, npg;      // first entry of the page table, pages
};

__device__ __forceinline__ SeqRows seq_rows(const Ragged& r, int b) {
  SeqRows s;
  if (r.qo_indptr) {
    s.row0 = min(max(gptr(r.qo_indptr)[b], 0), r.rows);
    s.n = min(max(gptr(r.qo_indptr)[b + 1], s.row0), r.rows) - s.row0;
  } else {
    s.row0 = b;
    s.n = 1;
  }
  s.len = min(max(gptr(r.kv_len)[b], 0), kMaxTokens);
  s.pg0 = min(max(gptr(r.kv_indptr)[b], 0), r.n_indices);
  s.npg = min(max(gptr(r.kv_indptr)[b + 1], s.pg0), r.n_indices) - s.pg0;
  return s;
}

// The sequence of row t: the last b with qo_indptr[b] <= t whose rows reach t
// (-1: behind the last sequence).  Uniform or per thread.
__device__ __forceinline__ int seq_of_row(const Ragged& r, int t) {
  if (!r.qo_indptr) return t < r.batch ? t : -1;
  int lo = 0, hi = r.batch;  // qo_indptr[lo] <= t < qo_indptr[hi] if t has a sequence
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (gptr(r.qo_indptr)[mid] <= t) lo = mid;
    else hi = mid;
  }
  return gptr(r.qo_indptr)[lo] <= t && t < gptr(r.qo_indptr)[hi] ? lo : -1;
}

// Device id of entry u of a sequence's page table, -1 where it has none.
__device__ __forceinline__ int page_id(const Ragged& r, const SeqRows& s, int u) {
  if (u < 0 || u >= s.npg) return -1;
  const int id = gptr(r.kv_indices)[s.pg0 + u];
  return (unsigned)id < (unsigned)r.num_pages ? id : -1;
}

// Tile `tile` of a batch cut into tiles of up to `rows` rows of one sequence ->
// {sequence (batch: none), its first row within the sequence}.  One thread, one
// sequence after another: 512 sequences of one row take the attention 436 us for 371
// without qo_indptr.
__device__ __forceinline__ void find_tile(const Ragged& r, int tile, int rows, int* out) {
  int b = tile, left = 0;
  if (r.qo_indptr) {
    left = tile;
    for (b = 0; b < r.batch; b++) {
      const int n = (seq_rows(r, b).n + rows - 1) / rows;
      if (left < n) break;
      left -= n;
    }
  }
  out[0] = b;
  out[1] = left * rows;
}

// Host checks of the parts every such operator has.
int ragged_check(const char* nm, const Ragged& r, int hq, int hkv, int d, int dtype);

}  // namespace yr
