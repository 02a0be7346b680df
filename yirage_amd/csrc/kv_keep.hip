// Keeping the accepted path of a tree of drafted tokens: the path's tokens move to the
// front of the sequence's new slots, where the next step continues.
//
//   slot[first + j] = slot[first + path[j]], j = 0, 1, ..    (first = len - n)
//
// A path ascends, so path[j] >= j: a slot is written only once the tokens that stay
// behind it have been read.  One thread moves the same 16 bytes of every token of the
// path, up to 8 in flight, so that order is the program's.  Bound by latency: a few
// dependent loads (lengths, path, page ids, tokens): one path 4.8 us, of 5 entries as of 12.
// With 64 sequences depth counts, 6.3 us for paths of 5 and 9.2 for 8: more places, each of a
// page of its own, on their way at once.
#include "ragged.h"

namespace yr {

struct KeepArgs {
  Ragged r;
  uint8_t* kc;  // tokens of `bytes` bytes
  uint8_t* vc;
  uint8_t* ks;  // tokens of hkv bytes, or null
  uint8_t* vs;
  uint16_t* bounds;  // [pages][hkv][2][D], or null
  const int32_t* path;
  int32_t* len_out;
  int depth, hkv, d, bytes, pieces;  // path entries; 16-byte pieces of a token
};

constexpr int KEEP_THREADS = 256, KEEP_AHEAD = 8;

template <int DT>
__global__ __launch_bounds__(KEEP_THREADS) void keep_kernel(KeepArgs a) {
  const Ragged& r = a.r;
  const int b = blockIdx.x, i = blockIdx.y * KEEP_THREADS + threadIdx.x;
  const SeqRows s = seq_rows(r, b);
  const int32_t* const path = a.path + (size_t)b * a.depth;
  const int first = s.len - s.n;
  // what this thread moves: a piece of K, one of V, or a head's two scales
  const bool is_k = i < a.pieces, is_v = !is_k && i < 2 * a.pieces;
  const int head = i - 2 * a.pieces;
  const bool is_s = a.ks && head >= 0 && head < a.hkv;
  uint8_t* const cache = is_k ? a.kc + 16 * i : a.vc + 16 * (i - a.pieces);
  // (bounds: this thread's 8 channels of a page's smallest and largest keys)
  const bool bounded = a.bounds && is_k;
  uint16_t* bd = nullptr;
  float lo[8], hi[8];
  auto flush = [&]() __attribute__((always_inline)) {
    if (!bd) return;
    uint32_t l[4], h[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      l[u] = pack2<DT>(lo[2 * u], lo[2 * u + 1]);
      h[u] = pack2<DT>(hi[2 * u], hi[2 * u + 1]);
    }
    stg16(bd, make_uint4(l[0], l[1], l[2], l[3]));
    stg16(bd + a.d, make_uint4(h[0], h[1], h[2], h[3]));
  };
  int kept = 0, last = -1;
  bool more = true;
  while (more) {
    int n = 0, from[KEEP_AHEAD];
#pragma unroll
    for (int u = 0; u < KEEP_AHEAD; u++) from[u] = kept + u < a.depth ? gptr(path)[kept + u] : -1;
#pragma unroll
    for (int u = 0; u < KEEP_AHEAD; u++) {
      more = more && from[u] > last && from[u] < s.n;
      if (more) {
        last = from[u];
        n++;
      } else {
        from[u] = 0;
      }
    }
    // (a token without a place is neither read nor written)
    long long src[KEEP_AHEAD], dst[KEEP_AHEAD];
    int page[KEEP_AHEAD];
    uint4 x[KEEP_AHEAD];
    uint8_t sk[KEEP_AHEAD], sv[KEEP_AHEAD];
#pragma unroll
    for (int u = 0; u < KEEP_AHEAD; u++) {
      const int p = first + from[u], q = first + kept + u;
      const bool some = u < n && p >= 0 && q >= 0;
      const int up = some ? p / r.page : -1, uq = some ? q / r.page : -1;
      const int f = page_id(r, s, up);
      page[u] = page_id(r, s, uq);
      if (f < 0) page[u] = -1;
      src[u] = (long long)max(f, 0) * r.page + p - up * r.page;
      dst[u] = (long long)max(page[u], 0) * r.page + q - uq * r.page;
    }
#pragma unroll
    for (int u = 0; u < KEEP_AHEAD; u++) {
      if (page[u] < 0) continue;
      if (is_k || is_v) x[u] = ldg16(cache + src[u] * a.bytes);
      else if (is_s) {
        sk[u] = gptr(a.ks)[src[u] * a.hkv + head];
        sv[u] = gptr(a.vs)[src[u] * a.hkv + head];
      }
    }
#pragma unroll
    for (int u = 0; u < KEEP_AHEAD; u++) {
      if (page[u] < 0) continue;
      if (is_k || is_v) {
        if (src[u] != dst[u]) stg16(cache + dst[u] * a.bytes, x[u]);
      } else if (is_s) {
        gptr(a.ks)[dst[u] * a.hkv + head] = sk[u];
        gptr(a.vs)[dst[u] * a.hkv + head] = sv[u];
      }
      if (bounded) {
        uint16_t* const at = a.bounds + ((size_t)page[u] * a.hkv + i / (a.d / 8)) * 2 * a.d + i % (a.d / 8) * 8;
        if (at != bd) {
          flush();
          bd = at;
          const uint4 l = ldg16(bd), h = ldg16(bd + a.d);
          const uint32_t lw[4] = {l.x, l.y, l.z, l.w}, hw[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
          for (int c = 0; c < 4; c++) {
            lo[2 * c] = lo16<DT>(lw[c]);
            lo[2 * c + 1] = hi16<DT>(lw[c]);
            hi[2 * c] = lo16<DT>(hw[c]);
            hi[2 * c + 1] = hi16<DT>(hw[c]);
          }
        }
        const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
        for (int c = 0; c < 4; c++) {  // (NaN left out)
          lo[2 * c] = fminf(lo[2 * c], lo16<DT>(w[c]));
          lo[2 * c + 1] = fminf(lo[2 * c + 1], hi16<DT>(w[c]));
          hi[2 * c] = fmaxf(hi[2 * c], lo16<DT>(w[c]));
          hi[2 * c + 1] = fmaxf(hi[2 * c + 1], hi16<DT>(w[c]));
        }
      }
    }
    kept += n;
  }
  flush();
  if (i == 0) gptr(a.len_out)[b] = max(first + kept, 0);
}

}  // namespace yr

using namespace yr;

extern "C" int yr_hip_keep_kv_paged(void* k_cache, void* v_cache, void* k_scale, void* v_scale, void* page_bounds,
                                    const int32_t* path, int depth, const int32_t* qo_indptr, const int32_t* kv_indptr,
                                    const int32_t* kv_indices, int n_indices, const int32_t* kv_len, int32_t* len_out,
                                    int batch, int hkv, int d, int page_size, int num_pages, int dtype,
                                    void* stream) {
  const char* nm = "yr_hip_keep_kv_paged";
  KeepArgs a;
  // (no tensor has a row a new token here: qo_indptr only says how many a sequence has)
  a.r = Ragged{qo_indptr, kv_indptr, kv_indices, kv_len, qo_indptr ? kMaxTokens : batch, batch, page_size, n_indices, num_pages};
  if (!k_cache || !v_cache || !path || !len_out) return fail(YR_E_INVALID, "%s: null pointer", nm);
  const bool e4m3 = dtype == YR_DTYPE_E4M3;
  if (e4m3 != (k_scale != nullptr) || e4m3 != (v_scale != nullptr))
    return fail(YR_E_INVALID, "%s: a cache in e4m3 comes with its scales, one in 16 bits without", nm);
  if (e4m3 && page_bounds) return fail(YR_E_INVALID, "%s: page bounds go with a cache in 16 bits", nm);
  int rc = ragged_check(nm, a.r, 0, hkv, d, e4m3 ? YR_DTYPE_BF16 : dtype);
  if (rc != YR_OK) return rc;
  if (depth < 1) return fail(YR_E_INVALID, "%s: a path has at least one entry", nm);
  if (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)page_bounds) & 15)
    return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  // (sequences are read and written in any order)
  const intptr_t apart = (intptr_t)len_out - (intptr_t)kv_len, size = (intptr_t)batch * (intptr_t)sizeof(int32_t);
  if (apart < size && -apart < size) return fail(YR_E_INVALID, "%s: the new lengths need a place of their own", nm);
  if (hkv > 1 << 20) return fail(YR_E_INVALID, "%s: too many heads", nm);
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.ks = (uint8_t*)k_scale;
  a.vs = (uint8_t*)v_scale;
  a.bounds = (uint16_t*)page_bounds;
  a.path = path;
  a.len_out = len_out;
  a.depth = depth;
  a.hkv = hkv;
  a.d = d;
  a.bytes = hkv * d * (e4m3 ? 1 : 2);
  a.pieces = a.bytes / 16;
  const int per = 2 * a.pieces + (e4m3 ? hkv : 0);
  const dim3 grid((unsigned)batch, (unsigned)((per + KEEP_THREADS - 1) / KEEP_THREADS));
  if (grid.y > 65535) return fail(YR_E_INVALID, "%s: too many heads", nm);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == YR_DTYPE_F16) hipLaunchKernelGGL((keep_kernel<DT_F16>), grid, dim3(KEEP_THREADS), 0, st, a);
  else hipLaunchKernelGGL((keep_kernel<DT_BF16>), grid, dim3(KEEP_THREADS), 0, st, a);
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
