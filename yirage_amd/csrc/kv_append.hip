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
//
// Bound by memory: every byte of q, k and v is read once and written once.  The
// angles are what else there is to read, in fp32 four times a q row's bytes, so a
// lane keeps them for 4 heads of its token (a row a lane: 97 us; two: 61; four
// 54; eight 72 for registers).  A page's keys and bounds belong to one workgroup
// and are reduced there, two channels a thread (a row's lanes alone: 88 us), and
// the stores pass the caches (kept in them: 69 us).  12.3k rows of 32 and 8 heads
// of 128 in bf16, 307 MB: 54 us, 5.6 TB/s, a copy of that size 58; 64 sequences'
// new tokens 5.5 us, one's 4.
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
  int hq, hkv, max_pos, q_blocks, q_chunks, heads;  // q_chunks per token; kv heads per cache workgroup
  float eps;
};

constexpr int AP_THREADS = 256;
constexpr int AP_WAVES = AP_THREADS / kWave;
constexpr int AP_Q = 4;  // q rows of a lane: they share its 32 angles

// A row (one token's head) is D / 16 lanes; a lane holds 8 elements of each
// half, so a rotated pair sits in one lane.
// What is written is not read again here: stored past the caches.
__device__ __forceinline__ void stg16_stream(uint16_t* p, uint4 v) {
  __builtin_nontemporal_store(__builtin_bit_cast(yr_u32x4, v), (YR_G yr_u32x4*)p);
}
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

// One lane's angles at position p.
template <int DT, int D, bool F32>
__device__ __forceinline__ void angles(const AppendArgs& a, int p, int l, float* c, float* s) {
  const size_t at = (size_t)p * D + 8 * l;
  table8<DT, F32>(a.cos, at, c);
  table8<DT, F32>(a.cos, at + D / 2, c + 8);
  table8<DT, F32>(a.sin, at, s);
  table8<DT, F32>(a.sin, at + D / 2, s + 8);
}

// One lane's 16 elements of a row, normalised by the weights w and rotated.
template <int DT, int D>
__device__ __forceinline__ void norm_rotate(bool norm, bool rotate, float eps, const float* w, const float* c,
                                            const float* s, uint4 lo, uint4 hi, uint4* out) {
  float x[16];
  unpack8<DT>(lo, x);
  unpack8<DT>(hi, x + 8);
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = 1; o < D / 16; o <<= 1) ss += __shfl_xor(ss, o, kWave);
    const float f = 1.f / sqrtf(ss * (1.f / D) + eps);
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = x[i] * f * w[i];
  }
  if (rotate) {
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
  constexpr int LPR = D / 16, RPW = kWave / LPR, RPP = AP_THREADS / LPR;  // lanes per row, rows per wave and per pass
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int l = tid % LPR, slot = tid / LPR;
  const Ragged& r = a.r;

  // ---- q: a wave takes AP_Q * RPW heads of one token
  if ((int)blockIdx.x < a.q_blocks) {
    const long long i = (long long)blockIdx.x * AP_WAVES + wave;
    const int t = (int)(i / a.q_chunks), h0 = (int)(i % a.q_chunks) * AP_Q * RPW + lane / LPR, g = a.hq / a.hkv;
    if (t >= r.rows) return;
    uint4 x[AP_Q][2];
#pragma unroll
    for (int j = 0; j < AP_Q; j++) {
      const int h = min(h0 + j * RPW, a.hq - 1);
      const uint16_t* src = a.q + t * a.q_row + (h / g) * a.q_grp + (h % g) * a.q_head + 8 * l;
      x[j][0] = ldg16(src);
      x[j][1] = ldg16(src + D / 2);
    }
    float w[16], c[16], sn[16];
    if (a.q_norm) {
      unpack8<DT>(ldg16(a.q_norm + 8 * l), w);
      unpack8<DT>(ldg16(a.q_norm + D / 2 + 8 * l), w + 8);
    }
    const int b = seq_of_row(r, t);
    if (b < 0) return;
    const SeqRows s = seq_rows(r, b);
    const int p = s.len - s.n + (t - s.row0);
    const bool lost = a.cos && (unsigned)p >= (unsigned)a.max_pos;  // no angle for this position: a loud answer
    if (a.cos && !lost) angles<DT, D, F32>(a, p, l, c, sn);
#pragma unroll
    for (int j = 0; j < AP_Q; j++) {
      const int h = h0 + j * RPW;
      if (h0 - lane / LPR + j * RPW >= a.hq) break;  // (uniform)
      uint4 y[2];
      norm_rotate<DT, D>(a.q_norm, a.cos, a.eps, w, c, sn, x[j][0], x[j][1], y);
      if (lost) {
        const uint32_t nan2 = pack2<DT>(NAN, NAN);
        y[0] = y[1] = make_uint4(nan2, nan2, nan2, nan2);
      }
      if (h < a.hq) {
        uint16_t* dst = a.q_out + ((size_t)t * a.hq + h) * D + 8 * l;
        stg16_stream(dst, y[0]);
        stg16_stream(dst + D / 2, y[1]);
      }
    }
    return;
  }

  // ---- k, v and bounds: one page of one sequence, a.heads kv heads
  const int groups = (a.hkv + a.heads - 1) / a.heads;
  const int item = (blockIdx.x - a.q_blocks) / groups, h0 = (blockIdx.x - a.q_blocks) % groups * a.heads;
  int b = item, u = 0;
  if (r.qo_indptr) {  // 64 sequences at a time, each wave for itself
    int left = item;
    for (b = 0; b < r.batch; b += kWave) {
      int pages = 0, p0 = 0;
      if (b + lane < r.batch) {
        const SeqRows s = seq_rows(r, b + lane);
        p0 = max(s.len - s.n, 0);
        pages = s.len > p0 ? (s.len - 1) / r.page - p0 / r.page + 1 : 0;
      }
      int sum = pages;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int v = __shfl_up(sum, o);
        if (lane >= o) sum += v;
      }
      const uint64_t past = __ballot(sum > left);
      if (past) {
        const int i = __builtin_ctzll(past);
        b += i;
        u = __builtin_amdgcn_readlane(p0 / r.page + left - (sum - pages), i);
        break;
      }
      left -= __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    if (b >= r.batch) return;
  }
  const SeqRows s = seq_rows(r, b);
  if (!r.qo_indptr) u = max(s.len - 1, 0) / r.page;
  const int id = page_id(r, s, u);
  if (id < 0) return;
  const int first = s.len - s.n;  // position of the sequence's first new row
  const int pos0 = max(max(first, 0), u * r.page);
  const int pos1 = min(min(s.len, (u + 1) * r.page), a.cos ? a.max_pos : 0x7fffffff);  // none without an angle
  if (pos0 >= pos1) return;
  const int hh = slot % a.heads, h = h0 + hh, step = RPP / a.heads;
  // the thread's word of the page's bounds, two channels (a head's first D / 2 words
  // are minima), as the tokens before left it
  const int word = tid % D;
  const bool low = word < D / 2;
  uint32_t* bd = nullptr;
  uint32_t old = low ? pack2<DT>(INFINITY, INFINITY) : pack2<DT>(-INFINITY, -INFINITY);
  if (a.bounds && tid / D < a.heads && h0 + tid / D < a.hkv) {
    bd = (uint32_t*)(a.bounds + ((size_t)id * a.hkv + h0 + tid / D) * 2 * D) + word;
    if (pos0 > u * r.page) old = gptr(bd)[0];
  }
  float mn[16], mx[16];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    mn[i] = INFINITY;
    mx[i] = -INFINITY;
  }
  if (h < a.hkv) {
    float w[16];
    if (a.k_norm) {
      unpack8<DT>(ldg16(a.k_norm + 8 * l), w);
      unpack8<DT>(ldg16(a.k_norm + D / 2 + 8 * l), w + 8);
    }
    for (int p = pos0 + slot / a.heads; p < pos1; p += step) {
      const long long t = s.row0 + (p - first);
      const uint16_t* ks = a.k + t * a.k_row + h * a.k_head + 8 * l;
      const uint16_t* vs = a.v + t * a.v_row + h * a.v_head + 8 * l;
      const uint4 v0 = ldg16(vs), v1 = ldg16(vs + D / 2);
      const uint4 k0 = ldg16(ks), k1 = ldg16(ks + D / 2);
      float c[16], sn[16];
      if (a.cos) angles<DT, D, F32>(a, p, l, c, sn);
      uint4 y[2];
      norm_rotate<DT, D>(a.k_norm, a.cos, a.eps, w, c, sn, k0, k1, y);
      const size_t dst = (((size_t)id * r.page + (p - u * r.page)) * a.hkv + h) * D + 8 * l;
      stg16_stream(a.kc + dst, y[0]);
      stg16_stream(a.kc + dst + D / 2, y[1]);
      stg16_stream(a.vc + dst, v0);
      stg16_stream(a.vc + dst + D / 2, v1);
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
  const int slots = min(RPP, (pos1 - pos0) * a.heads);
  if (slot < slots) {
    s_b[slot][0][l] = pack8<DT>(mn);
    s_b[slot][1][l] = pack8<DT>(mn + 8);
    s_b[slot][2][l] = pack8<DT>(mx);
    s_b[slot][3][l] = pack8<DT>(mx + 8);
  }
  __syncthreads();
  float e0 = lo16<DT>(old), e1 = hi16<DT>(old);
  const uint32_t* const rows = (const uint32_t*)s_b + word;
#pragma unroll 8
  for (int o = tid / D; o < slots; o += a.heads) {
    const uint32_t x = rows[o * D];
    e0 = low ? fminf(e0, lo16<DT>(x)) : fmaxf(e0, lo16<DT>(x));
    e1 = low ? fminf(e1, hi16<DT>(x)) : fmaxf(e1, hi16<DT>(x));
  }
  if (bd) gptr(bd)[0] = pack2<DT>(e0, e1);
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
  const int rpp = AP_THREADS / (d / 16), chunk = AP_Q * kWave / (d / 16);
  a.q_chunks = ((q ? hq : 1) + chunk - 1) / chunk;
  const long long qb = q ? ((long long)rows * a.q_chunks + AP_WAVES - 1) / AP_WAVES : 0;
  // pages that new rows can touch: each sequence's span, at most one per row
  long long items = (long long)rows / page_size + 2ll * batch;
  if (items > rows) items = rows;
  // kv heads per workgroup: as many as leave every row slot a token of the page and
  // each thread one word of the bounds
  const int tokens = qo_indptr ? (int)((rows + batch - 1) / batch < page_size ? (rows + batch - 1) / batch : page_size) : 1;
  a.heads = 1;
  while (a.heads < hkv && a.heads * tokens < rpp && a.heads < AP_THREADS / d) a.heads *= 2;
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
