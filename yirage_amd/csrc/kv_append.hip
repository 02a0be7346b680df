// Appending new tokens to a paged key-value cache: k (and q) are normalised per
// head (optional), rotated by their position and rounded once, k and v go to
// their slots, and every page keeps the smallest and largest stored key per
// channel and kv head (page_bounds), the summary that page selection scores.
//
//   y[d] = x[d] cos[p][d] - x[d + D/2] sin[p][d]        (d < D/2)
//   y[d] = x[d] cos[p][d] + x[d - D/2] sin[p][d]        (d >= D/2)
//   x = raw * rsqrt(mean(raw^2) + eps) * w              (with norm weights)
//
// All of it in fp32 from 16-bit inputs, rounded once to the cache's type; the
// bounds are taken of the rounded keys, so they are exact.
#include "ragged.h"

namespace yr {

struct AppendArgs {
  Ragged r;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  uint16_t* kc;
  uint16_t* vc;
  uint16_t* bounds;  // [pages][hkv][2][D]
  const void* cos;
  const void* sin;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  long long q_row, q_grp, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int hq, hkv, max_pos, q_blocks, heads;  // heads: kv heads per cache workgroup
  float eps;
};

constexpr int AP_THREADS = 256;

// A row (one token's head) is D / 16 lanes; a lane holds 8 elements of each
// half, so a rotated pair sits in one lane.
template <int DT>
__device__ __forceinline__ void unpack8(uint4 v, float* x) {
  x[0] = lo16<DT>(v.x); x[1] = hi16<DT>(v.x); x[2] = lo16<DT>(v.y); x[3] = hi16<DT>(v.y);
  x[4] = lo16<DT>(v.z); x[5] = hi16<DT>(v.z); x[6] = lo16<DT>(v.w); x[7] = hi16<DT>(v.w);
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7]));
}

// 8 table entries at `at`
template <int DT, bool F32>
__device__ __forceinline__ void table8(const void* t, size_t at, float* x) {
  if constexpr (F32) {
    const uint4 a = ldg16((const float*)t + at), b = ldg16((const float*)t + at + 4);
    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
  } else {
    unpack8<DT>(ldg16((const uint16_t*)t + at), x);
  }
}

// One lane's 16 elements of a row, normalised and rotated for position p.
template <int DT, int D, bool F32>
__device__ __forceinline__ void norm_rotate(const AppendArgs& a, const uint16_t* w, uint4 lo, uint4 hi, int p, int l,
                                            uint4* out) {
  float x[16];
  unpack8<DT>(lo, x);
  unpack8<DT>(hi, x + 8);
  if (w) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = 1; o < D / 16; o <<= 1) ss += __shfl_xor(ss, o, kWave);
    const float f = 1.f / sqrtf(ss * (1.f / D) + a.eps);
    float wv[16];
    unpack8<DT>(ldg16(w + 8 * l), wv);
    unpack8<DT>(ldg16(w + D / 2 + 8 * l), wv + 8);
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = x[i] * f * wv[i];
  }
  if (a.cos) {
    float c[16], s[16];
    const size_t at = (size_t)p * D + 8 * l;
    table8<DT, F32>(a.cos, at, c);
    table8<DT, F32>(a.cos, at + D / 2, c + 8);
    table8<DT, F32>(a.sin, at, s);
    table8<DT, F32>(a.sin, at + D / 2, s + 8);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float u = x[i], t = x[i + 8];
      x[i] = u * c[i] - t * s[i];
      x[i + 8] = t * c[i + 8] + u * s[i + 8];
    }
  }
  out[0] = pack8<DT>(x);
  out[1] = pack8<DT>(x + 8);
}

template <int DT, int D, bool F32>
__global__ __launch_bounds__(AP_THREADS) void append_kernel(AppendArgs a) {
  constexpr int LPR = D / 16, RPP = AP_THREADS / LPR;  // lanes per row, rows per pass
  const int tid = threadIdx.x, l = tid % LPR, slot = tid / LPR;
  const Ragged& r = a.r;

  // ---- q: rows of (token, head)
  if ((int)blockIdx.x < a.q_blocks) {
    const long long i = (long long)blockIdx.x * RPP + slot;
    const int t = (int)(i / a.hq), h = (int)(i % a.hq), g = a.hq / a.hkv;
    if (t >= r.rows) return;
    const int b = seq_of_row(r, t);
    if (b < 0) return;
    const SeqRows s = seq_rows(r, b);
    const int p = s.len - s.n + (t - s.row0);
    const uint16_t* src = a.q + t * a.q_row + (h / g) * a.q_grp + (h % g) * a.q_head + 8 * l;
    uint4 y[2];
    if (a.cos && (unsigned)p >= (unsigned)a.max_pos) {  // no angle for this position: a loud answer
      const uint32_t nan2 = pack2<DT>(NAN, NAN);
      y[0] = y[1] = make_uint4(nan2, nan2, nan2, nan2);
    } else {
      norm_rotate<DT, D, F32>(a, a.q_norm, ldg16(src), ldg16(src + D / 2), p, l, y);
    }
    uint16_t* dst = a.q_out + ((size_t)t * a.hq + h) * D + 8 * l;
    stg16(dst, y[0]);
    stg16(dst + D / 2, y[1]);
    return;
  }

  // ---- k, v and bounds: one page of one sequence, a.heads kv heads
  const int groups = (a.hkv + a.heads - 1) / a.heads;
  const int item = (blockIdx.x - a.q_blocks) / groups, h0 = (blockIdx.x - a.q_blocks) % groups * a.heads;
  __shared__ int s_item[2];
  if (tid == 0) {
    int left = item, b = 0, u = -1;
    for (; b < r.batch; b++) {
      const SeqRows s = seq_rows(r, b);
      const int p0 = max(s.len - s.n, 0);
      const int pages = s.len > p0 ? (s.len - 1) / r.page - p0 / r.page + 1 : 0;
      if (left < pages) {
        u = p0 / r.page + left;
        break;
      }
      left -= pages;
    }
    s_item[0] = b;
    s_item[1] = u;
  }
  __syncthreads();
  const int b = s_item[0], u = s_item[1];
  if (u < 0) return;
  const SeqRows s = seq_rows(r, b);
  const int id = page_id(r, s, u);
  if (id < 0) return;
  const int first = s.len - s.n;  // position of the sequence's first new row
  const int pos0 = max(max(first, 0), u * r.page);
  const int pos1 = min(min(s.len, (u + 1) * r.page), a.cos ? a.max_pos : 0x7fffffff);  // none without an angle
  if (pos0 >= pos1) return;
  const int hh = slot % a.heads, h = h0 + hh, step = RPP / a.heads;
  float mn[16], mx[16];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    mn[i] = INFINITY;
    mx[i] = -INFINITY;
  }
  if (h < a.hkv) {
    for (int p = pos0 + slot / a.heads; p < pos1; p += step) {
      const long long t = s.row0 + (p - first);
      const uint16_t* ks = a.k + t * a.k_row + h * a.k_head + 8 * l;
      const uint16_t* vs = a.v + t * a.v_row + h * a.v_head + 8 * l;
      const uint4 v0 = ldg16(vs), v1 = ldg16(vs + D / 2);
      uint4 y[2];
      norm_rotate<DT, D, F32>(a, a.k_norm, ldg16(ks), ldg16(ks + D / 2), p, l, y);
      const size_t dst = (((size_t)id * r.page + (p - u * r.page)) * a.hkv + h) * D + 8 * l;
      stg16(a.kc + dst, y[0]);
      stg16(a.kc + dst + D / 2, y[1]);
      stg16(a.vc + dst, v0);
      stg16(a.vc + dst + D / 2, v1);
      float x[16];
      unpack8<DT>(y[0], x);
      unpack8<DT>(y[1], x + 8);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        mn[i] = fminf(mn[i], x[i]);
        mx[i] = fmaxf(mx[i], x[i]);
      }
    }
  }
  if (!a.bounds) return;
  __shared__ uint4 s_b[RPP][4][LPR];
  s_b[slot][0][l] = pack8<DT>(mn);
  s_b[slot][1][l] = pack8<DT>(mn + 8);
  s_b[slot][2][l] = pack8<DT>(mx);
  s_b[slot][3][l] = pack8<DT>(mx + 8);
  __syncthreads();
  if (slot >= a.heads || h >= a.hkv) return;
  for (int o = slot + a.heads; o < RPP; o += a.heads) {
    float x[16];
    unpack8<DT>(s_b[o][0][l], x);
    unpack8<DT>(s_b[o][1][l], x + 8);
#pragma unroll
    for (int i = 0; i < 16; i++) mn[i] = fminf(mn[i], x[i]);
    unpack8<DT>(s_b[o][2][l], x);
    unpack8<DT>(s_b[o][3][l], x + 8);
#pragma unroll
    for (int i = 0; i < 16; i++) mx[i] = fmaxf(mx[i], x[i]);
  }
  uint16_t* bd = a.bounds + ((size_t)id * a.hkv + h) * 2 * D + 8 * l;
  if (pos0 > u * r.page) {  // the page held tokens already
    float x[16];
    unpack8<DT>(ldg16(bd), x);
    unpack8<DT>(ldg16(bd + D / 2), x + 8);
#pragma unroll
    for (int i = 0; i < 16; i++) mn[i] = fminf(mn[i], x[i]);
    unpack8<DT>(ldg16(bd + D), x);
    unpack8<DT>(ldg16(bd + D + D / 2), x + 8);
#pragma unroll
    for (int i = 0; i < 16; i++) mx[i] = fmaxf(mx[i], x[i]);
  }
  stg16(bd, pack8<DT>(mn));
  stg16(bd + D / 2, pack8<DT>(mn + 8));
  stg16(bd + D, pack8<DT>(mx));
  stg16(bd + D + D / 2, pack8<DT>(mx + 8));
}

int ragged_check(const char* nm, const Ragged& r, int hq, int hkv, int d, int dtype) {
  if (!r.kv_indptr || !r.kv_indices || !r.kv_len) return fail(YR_E_INVALID, "%s: null pointer", nm);
  if (dtype != YR_DTYPE_F16 && dtype != YR_DTYPE_BF16) return fail(YR_E_INVALID, "%s: dtype", nm);
  if (d != 64 && d != 128) return fail(YR_E_INVALID, "%s: head_dim %d unsupported (64, 128)", nm, d);
  if (r.rows <= 0 || r.batch <= 0) return fail(YR_E_INVALID, "%s: rows and batch must be positive", nm);
  if (hkv <= 0 || hq < 0 || hq % hkv) return fail(YR_E_INVALID, "%s: hq must be a multiple of hkv", nm);
  if (r.page <= 0 || r.page > kMaxPage || r.num_pages <= 0 || r.n_indices < 0) return fail(YR_E_INVALID, "%s: bad page size or count", nm);
  if (!r.qo_indptr && r.rows != r.batch)
    return fail(YR_E_INVALID, "%s: without qo_indptr every sequence has one row (%d rows, batch %d)", nm, r.rows, r.batch);
  return YR_OK;
}

}  // namespace yr

using namespace yr;

extern "C" int yr_hip_append_kv_paged(const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                                      void* v_cache, void* page_bounds, const void* cos_table, const void* sin_table,
                                      int table_dtype, int max_pos, const void* q_norm, const void* k_norm, float eps,
                                      const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                                      int n_indices, const int32_t* kv_len, int rows, int batch, int hq, int hkv, int d,
                                      int page_size, int num_pages, const int64_t* strides7, int dtype, void* stream) {
  const char* nm = "yr_hip_append_kv_paged";
  AppendArgs a;
  a.r = Ragged{qo_indptr, kv_indptr, kv_indices, kv_len, rows, batch, page_size, n_indices, num_pages};
  if (!k || !v || !k_cache || !v_cache || !strides7) return fail(YR_E_INVALID, "%s: null pointer", nm);
  if (!q != !q_out) return fail(YR_E_INVALID, "%s: q and q_out come together", nm);
  if (!cos_table != !sin_table) return fail(YR_E_INVALID, "%s: cos and sin come together", nm);
  int rc = ragged_check(nm, a.r, q ? hq : 0, hkv, d, dtype);
  if (rc != YR_OK) return rc;
  if (q && hq <= 0) return fail(YR_E_INVALID, "%s: hq must be positive", nm);
  if (cos_table && ((table_dtype != YR_DTYPE_F32 && table_dtype != dtype) || max_pos <= 0))
    return fail(YR_E_INVALID, "%s: tables are fp32 or of k's type, with at least one position", nm);
  uintptr_t low = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_cache |
                  (uintptr_t)v_cache | (uintptr_t)page_bounds | (uintptr_t)cos_table | (uintptr_t)sin_table |
                  (uintptr_t)q_norm | (uintptr_t)k_norm;
  if (low & 15) return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  for (int i = q ? 0 : 3; i < 7; i++)
    if (strides7[i] % 8) return fail(YR_E_INVALID, "%s: strides must be multiples of 8 elements", nm);
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.q_out = (uint16_t*)q_out;
  a.kc = (uint16_t*)k_cache;
  a.vc = (uint16_t*)v_cache;
  a.bounds = (uint16_t*)page_bounds;
  a.cos = cos_table;
  a.sin = sin_table;
  a.q_norm = (const uint16_t*)q_norm;
  a.k_norm = (const uint16_t*)k_norm;
  a.q_row = strides7[0];
  a.q_grp = strides7[1];
  a.q_head = strides7[2];
  a.k_row = strides7[3];
  a.k_head = strides7[4];
  a.v_row = strides7[5];
  a.v_head = strides7[6];
  a.hq = q ? hq : hkv;
  a.hkv = hkv;
  a.max_pos = max_pos;
  a.eps = eps;
  const int rpp = AP_THREADS / (d / 16);
  const long long qb = q ? ((long long)rows * hq + rpp - 1) / rpp : 0;
  // pages that new rows can touch: each sequence's span, at most one per row
  long long items = (long long)rows / page_size + 2ll * batch;
  if (items > rows) items = rows;
  // kv heads per workgroup: as many as leave every row slot a token of the page
  const int tokens = qo_indptr ? (int)((rows + batch - 1) / batch < page_size ? (rows + batch - 1) / batch : page_size) : 1;
  a.heads = 1;
  while (a.heads < hkv && a.heads * tokens < rpp && a.heads < rpp) a.heads *= 2;
  const long long blocks = qb + items * ((hkv + a.heads - 1) / a.heads);
  if (blocks > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
  a.q_blocks = (int)qb;
  const bool f32 = table_dtype == YR_DTYPE_F32;
  hipStream_t st = (hipStream_t)stream;
#define YR_AP(DT_, D_, F_)                                                                                     \
  if (dtype == DT_ && d == D_ && f32 == F_)                                                                    \
    hipLaunchKernelGGL((append_kernel<DT_, D_, F_>), dim3((unsigned)blocks), dim3(AP_THREADS), 0, st, a);
  YR_AP(DT_F16, 64, false) YR_AP(DT_F16, 64, true) YR_AP(DT_F16, 128, false) YR_AP(DT_F16, 128, true)
  YR_AP(DT_BF16, 64, false) YR_AP(DT_BF16, 64, true) YR_AP(DT_BF16, 128, false) YR_AP(DT_BF16, 128, true)
#undef YR_AP
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
