// Selecting the pages of a long cache that a query row attends to, by an upper
// bound of its scores.  With min / max the smallest and largest key of page u
// per channel (kv_append.hip keeps them),
//
//   sum over tokens' best case = sum_g sum_d max(q_gd min_ud, q_gd max_ud)
//                              = sum_d Q+_d max_ud + Q-_d min_ud,
//   Q+ = sum over the group's heads of max(q, 0), Q- = sum of min(q, 0),
//
// so a page costs 2 D products per (row, kv head) whatever the group size.  A
// row takes its first `first` pages, its last `last` visible ones and the best
// bounds among the rest, ties to the lower page, and lists them in order.
//
// The sums run in 64 bits: 16-bit factors are exact there, and the border
// between the last page taken and the first one left is often narrower than
// 32-bit rounding, which would make the list depend on the order of the sum.
#include "ragged.h"

namespace yr {

struct SelectArgs {
  Ragged r;
  const uint16_t* q;
  const uint16_t* bounds;  // [pages][hkv][2][D]
  int32_t* out;            // [rows][hkv][top]
  int hq, hkv, max_pages, top, first, last;
};

constexpr int SEL_THREADS = 256;
constexpr int SEL_WAVES = SEL_THREADS / kWave;
constexpr int SEL_MAX_PAGES = 16384;  // 64-bit keys of one row in LDS: 128 of 160 KiB

// Whole-number order of a score: larger is better, -0 equals 0, NaN is last.
__device__ __forceinline__ uint64_t score_key(double s) {
  if (s != s) return 0;
  const int64_t b = __double_as_longlong(s + 0.0);
  return b < 0 ? ~(uint64_t)b : (uint64_t)b | 0x8000000000000000ull;
}

// Writes the ascending list of a row: pages [0, f) and [n - l, n) and the `m`
// best keys of [f, n - l), -1 behind.  Called by the whole workgroup.
__device__ void choose(const uint64_t* key, int n, int f, int l, int m, int top, int32_t* out) {
  __shared__ int s_hist[256];
  __shared__ uint64_t s_lo;
  __shared__ int s_need, s_done, s_cnt[SEL_WAVES][2];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int c0 = f, c1 = n - l;  // candidates
  // Radix selection, 8 bits at a time: `lo` is the m-th best key's known prefix,
  // `need` how many of the keys with that prefix are still to be taken.
  uint64_t lo = 0;
  int need = m;
  bool exact = false;  // `need` of the keys equal to lo, not all keys from lo on
  if (m > 0 && m < c1 - c0) {
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SEL_THREADS) s_hist[i] = 0;
      __syncthreads();
      for (int u = c0 + tid; u < c1; u += SEL_THREADS) {
        const uint64_t k = key[u];
        if (shift == 56 || (k >> (shift + 8)) == (lo >> (shift + 8))) atomicAdd(&s_hist[(int)(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = need, bin = 255;
        for (; bin > 0 && s_hist[bin] < left; bin--) left -= s_hist[bin];
        s_lo = lo | ((uint64_t)bin << shift);
        s_need = left;
        s_done = s_hist[bin] == left;  // the whole bin is taken
      }
      __syncthreads();
      lo = s_lo;
      need = s_need;
      const bool done = s_done;
      __syncthreads();
      if (done) break;
      exact = shift == 0;
    }
  }
  // ascending list
  int at = 0, eq = 0;  // written so far, keys equal to lo seen so far
  for (int u0 = 0; u0 < n; u0 += SEL_THREADS) {
    const int u = u0 + tid;
    const bool cand = u >= c0 && u < c1;
    const uint64_t k = cand ? key[u] : 0;
    const bool same = exact && cand && k == lo;
    const uint64_t be = __ballot(same);
    if (lane == 0) s_cnt[wave][0] = __popcll(be);
    __syncthreads();
    int before = eq, alle = 0;
    for (int w = 0; w < SEL_WAVES; w++) {
      if (w < wave) before += s_cnt[w][0];
      alle += s_cnt[w][0];
    }
    before += __popcll(be & ((1ull << lane) - 1));
    const bool take = u < n && (!cand || (m > 0 && (same ? before < need : k >= lo)));
    const uint64_t bt = __ballot(take);
    if (lane == 0) s_cnt[wave][1] = __popcll(bt);
    __syncthreads();
    int pos = at, all = 0;
    for (int w = 0; w < SEL_WAVES; w++) {
      if (w < wave) pos += s_cnt[w][1];
      all += s_cnt[w][1];
    }
    pos += __popcll(bt & ((1ull << lane) - 1));
    if (take && pos < top) gptr(out)[pos] = u;
    at += all;
    eq += alle;
    __syncthreads();
  }
  for (int i = at + tid; i < top; i += SEL_THREADS) gptr(out)[i] = -1;
}

template <int DT, int D>
__global__ __launch_bounds__(SEL_THREADS) void select_kernel(SelectArgs a) {
  constexpr int LPP = D / 8, PPB = SEL_THREADS / LPP;  // lanes per page, pages per pass
  extern __shared__ uint64_t s_key[];
  __shared__ double s_q[2][D];
  const int h = blockIdx.x % a.hkv, t = blockIdx.x / a.hkv, tid = threadIdx.x;
  const int b = seq_of_row(a.r, t);
  if (b < 0) return;
  const SeqRows s = seq_rows(a.r, b);
  int32_t* out = a.out + ((size_t)t * a.hkv + h) * a.top;
  const int p = s.len - s.n + (t - s.row0);
  // visible pages that exist
  const int n = p < 0 ? 0 : min(min(p / a.r.page + 1, s.npg), a.max_pages);
  const int g = a.hq / a.hkv;
  for (int d = tid; d < D; d += SEL_THREADS) {
    double up = 0, down = 0;
    for (int i = 0; i < g; i++) {
      const double x = ld_elem<DT>(gptr(a.q)[((size_t)t * a.hq + (size_t)h * g + i) * D + d]);
      up += x > 0 ? x : 0;
      down += x < 0 ? x : 0;
    }
    s_q[0][d] = down;
    s_q[1][d] = up;
  }
  __syncthreads();
  const int f = min(a.first, n), l = min(a.last, n - f);
  const int m = min(max(a.top - f - l, 0), n - f - l);
  if (m > 0 && m < n - f - l) {
    const int j = tid % LPP;
    double qd[8], qu[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qd[i] = s_q[0][8 * j + i];
      qu[i] = s_q[1][8 * j + i];
    }
    for (int u0 = f; u0 < n - l; u0 += PPB) {
      const int u = u0 + tid / LPP;
      const int id = u < n - l ? page_id(a.r, s, u) : -1;
      double sum = 0;
      if (id >= 0) {
        const uint16_t* bd = a.bounds + ((size_t)id * a.hkv + h) * 2 * D + 8 * j;
        const uint4 mn = ldg16(bd), mx = ldg16(bd + D);
        const uint32_t w0[4] = {mn.x, mn.y, mn.z, mn.w}, w1[4] = {mx.x, mx.y, mx.z, mx.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          sum = fma(qd[2 * i], (double)lo16<DT>(w0[i]), sum);
          sum = fma(qd[2 * i + 1], (double)hi16<DT>(w0[i]), sum);
          sum = fma(qu[2 * i], (double)lo16<DT>(w1[i]), sum);
          sum = fma(qu[2 * i + 1], (double)hi16<DT>(w1[i]), sum);
        }
      }
#pragma unroll
      for (int o = 1; o < LPP; o <<= 1) sum += __shfl_xor(sum, o, kWave);
      if (j == 0 && u < n - l) s_key[u] = id < 0 ? 0 : score_key(sum);
    }
  }
  __syncthreads();
  choose(s_key, n, f, l, m, a.top, out);
}

}  // namespace yr

using namespace yr;

extern "C" int yr_hip_select_pages(const void* q, const void* page_bounds, const int32_t* qo_indptr,
                                   const int32_t* kv_indptr, const int32_t* kv_indices, int n_indices,
                                   const int32_t* kv_len, int32_t* pages, int rows, int batch, int hq, int hkv, int d,
                                   int page_size, int num_pages, int max_kv_len, int top_pages, int first_pages,
                                   int last_pages, int dtype, void* stream) {
  const char* nm = "yr_hip_select_pages";
  SelectArgs a;
  a.r = Ragged{qo_indptr, kv_indptr, kv_indices, kv_len, rows, batch, page_size, n_indices, num_pages};
  if (!q || !page_bounds || !pages) return fail(YR_E_INVALID, "%s: null pointer", nm);
  int rc = ragged_check(nm, a.r, hq, hkv, d, dtype);
  if (rc != YR_OK) return rc;
  if (hq <= 0) return fail(YR_E_INVALID, "%s: hq must be positive", nm);
  if (((uintptr_t)q | (uintptr_t)page_bounds) & 15) return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  if (max_kv_len <= 0) return fail(YR_E_INVALID, "%s: max_kv_len must be > 0", nm);
  if (first_pages < 0 || last_pages < 1) return fail(YR_E_INVALID, "%s: the last page at least is taken", nm);
  if (top_pages < 1 || (long long)first_pages + last_pages > top_pages)
    return fail(YR_E_INVALID, "%s: top_pages must cover first_pages + last_pages", nm);
  a.max_pages = (max_kv_len - 1) / page_size + 1;
  if (a.max_pages > SEL_MAX_PAGES)
    return fail(YR_E_INVALID, "%s: %d pages a sequence exceed %d (page_size too small)", nm, a.max_pages, SEL_MAX_PAGES);
  if ((long long)rows * hkv > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
  a.q = (const uint16_t*)q;
  a.bounds = (const uint16_t*)page_bounds;
  a.out = pages;
  a.hq = hq;
  a.hkv = hkv;
  a.top = top_pages;
  a.first = first_pages;
  a.last = last_pages;
  const size_t lds = (size_t)a.max_pages * 8;
  hipStream_t st = (hipStream_t)stream;
#define YR_SEL(DT_, D_)                                                                                             \
  if (dtype == DT_ && d == D_)                                                                                      \
    hipLaunchKernelGGL((select_kernel<DT_, D_>), dim3((unsigned)(rows * hkv)), dim3(SEL_THREADS), lds, st, a);
  YR_SEL(DT_F16, 64) YR_SEL(DT_F16, 128) YR_SEL(DT_BF16, 64) YR_SEL(DT_BF16, 128)
#undef YR_SEL
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
