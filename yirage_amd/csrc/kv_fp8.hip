// A paged key-value cache in 8 bits: e4m3 codes with a power of two per token and kv
// head (e8m0), written by the append and read back to 16 bits.
//
//   scale = 2^e, e the smallest (>= -126) with max |x| <= 448 2^e
//   code = x / scale rounded to e4m3, value = code scale
//
// A power of two costs a floating code nothing but range (a step is a part of the
// value, not of the scale), makes division and product exact, and is what the
// conversion instructions take.  x is the normalised, rotated key or the value in fp32:
// one rounding, half a step of e4m3 (2^-4 of the value; 2^-10 scale below 2^-6 scale).
// A head with a NaN or an infinity gets the scale NaN: it reads as NaN throughout.
#include <type_traits>

#include "kv_rows.h"

namespace yr {

struct Append8Args {
  Ragged r;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  uint8_t* kc;  // [pages][page][hkv][D]
  uint8_t* vc;
  uint8_t* ks;  // [pages][page][hkv]
  uint8_t* vs;
  const void* cos;
  const void* sin;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  const int32_t* positions;
  long long q_row, q_grp, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int hq, hkv, max_pos, chunks;  // hq 0 without q; waves per token
  float eps;
};

constexpr int A8_THREADS = 256;
constexpr int A8_ROWS = 4;  // rows of a lane

// 16 values of a row, shared by D / 16 lanes -> 8 codes of each half and the scale's byte.
template <int D>
__device__ __forceinline__ int quantise16(const float* x, uint2* codes) {
  uint32_t top = 0;  // as whole numbers NaN > infinity > finite
#pragma unroll
  for (int i = 0; i < 16; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < D / 16; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, kWave));
  codes[0] = codes[1] = make_uint2(0, 0);
  if (top >= 0x7f800000u) return 255;
  // top = m 2^k: 448 = 1.75 2^8 holds it at e = k - 8, or k - 7 where m > 1.75
  const int e = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u), -126);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const float* y = x + 8 * h;
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
    codes[h] = make_uint2((uint32_t)lo, (uint32_t)hi);
  }
  return e + 127;
}

// A wave takes up to A8_ROWS * RPW of a token's rows, q heads first, then k's and v's: its
// lanes keep the token's angles for all of theirs, and the search for the token's sequence and
// page runs while the rows are on their way.  12.4k tokens of 32 and 8 heads of 128 in bf16, 281 MB:
// 53 us, 5.3 TB/s, bound by memory (a copy of that size 55); one token 4.8 us, bound by latency.
// (The sequence searched for by all lanes at once instead of by halving: 56.5 us.)
template <int DT, int D, bool F32>
__global__ __launch_bounds__(A8_THREADS) void append8_kernel(Append8Args a) {
  constexpr int LPR = D / 16, RPW = kWave / LPR, WAVES = A8_THREADS / kWave;  // lanes per row, rows per wave and pass
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int l = lane % LPR;
  const Ragged& r = a.r;
  const long long item = (long long)blockIdx.x * WAVES + wave;
  const int t = (int)(item / a.chunks), row0 = (int)(item % a.chunks) * A8_ROWS * RPW, rows = a.hq + 2 * a.hkv;
  if (t >= r.rows) return;
  const int g = a.hq / a.hkv;
  uint4 x[A8_ROWS][2];
#pragma unroll
  for (int j = 0; j < A8_ROWS; j++) {
    const int i = min(row0 + j * RPW + lane / LPR, rows - 1);
    const uint16_t* src;
    if (i < a.hq) src = a.q + t * a.q_row + (i / g) * a.q_grp + (i % g) * a.q_head;
    else if (i < a.hq + a.hkv) src = a.k + t * a.k_row + (i - a.hq) * a.k_head;
    else src = a.v + t * a.v_row + (i - a.hq - a.hkv) * a.v_head;
    x[j][0] = ldg16(src + 8 * l);
    x[j][1] = ldg16(src + D / 2 + 8 * l);
  }
  const int b = seq_of_row(r, t);
  if (b < 0) return;
  const SeqRows s = seq_rows(r, b);
  const int p = s.len - s.n + (t - s.row0), at = a.positions ? gptr(a.positions)[t] : p;
  const bool lost = a.cos && (unsigned)at >= (unsigned)a.max_pos;  // no angle: q is NaN, the token is not written
  float c[16], sn[16];
  if (a.cos && !lost) angles<DT, D, F32>(a.cos, a.sin, at, l, c, sn);
  const int id = p < 0 || lost ? -1 : page_id(r, s, p / r.page);
  const size_t slot = ((size_t)max(id, 0) * r.page + max(p, 0) % r.page) * a.hkv;
#pragma unroll
  for (int j = 0; j < A8_ROWS; j++) {
    if (row0 + j * RPW >= rows) break;  // (uniform)
    const int i = row0 + j * RPW + lane / LPR;
    const bool is_q = i < a.hq, is_v = i >= a.hq + a.hkv;
    float y[16];
    unpack8<DT>(x[j][0], y);
    unpack8<DT>(x[j][1], y + 8);
    const uint16_t* const wt = is_q ? a.q_norm : a.k_norm;
    // every lane of the wave takes part in the row sums; values keep what they were
    if (a.q_norm || a.k_norm || a.cos) {
      float z[16], w[16];
#pragma unroll
      for (int u = 0; u < 16; u++) z[u] = y[u];
      if (a.q_norm || a.k_norm) {
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < 16; u++) ss = fmaf(z[u], z[u], ss);
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor(ss, o, kWave);
        if (wt && !is_v) {
          const float f = 1.f / sqrtf(ss * (1.f / D) + a.eps);
          unpack8<DT>(ldg16(wt + 8 * l), w);
          unpack8<DT>(ldg16(wt + D / 2 + 8 * l), w + 8);
#pragma unroll
          for (int u = 0; u < 16; u++) z[u] = z[u] * f * w[u];
        }
      }
      norm_rotate<D>(false, a.cos, 0.f, w, c, sn, z);
#pragma unroll
      for (int u = 0; u < 16; u++) y[u] = is_v ? y[u] : z[u];
    }
    uint2 codes[2];
    const int scale = quantise16<D>(y, codes);
    if (is_q) {
      uint4 o[2] = {pack8<DT>(y), pack8<DT>(y + 8)};
      if (lost) {
        const uint32_t nan2 = pack2<DT>(NAN, NAN);
        o[0] = o[1] = make_uint4(nan2, nan2, nan2, nan2);
      }
      uint16_t* dst = a.q_out + ((size_t)t * a.hq + i) * D + 8 * l;
      stg16_stream(dst, o[0]);
      stg16_stream(dst + D / 2, o[1]);
    } else if (i < rows && id >= 0) {
      const size_t head = slot + (is_v ? i - a.hq - a.hkv : i - a.hq);
      uint8_t* const dst = (is_v ? a.vc : a.kc) + head * D + 8 * l;
      *(YR_G uint64_t*)dst = (uint64_t)codes[0].y << 32 | codes[0].x;
      *(YR_G uint64_t*)(dst + D / 2) = (uint64_t)codes[1].y << 32 | codes[1].x;
      if (l == 0) gptr(is_v ? a.vs : a.ks)[head] = (uint8_t)scale;
    }
  }
}

struct Read8Args {
  Ragged r;  // qo_indptr: rows of the result, from each sequence's first token on
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  uint16_t* k;  // [rows][hkv][D]
  uint16_t* v;
  int hkv;
};

// 8 codes and their scale -> 8 values of 16 bits.  Exact in bf16 wherever the value
// is normal, rounded once in f16; a scale of NaN gives NaN.
template <int DT>
__device__ __forceinline__ uint4 values8(uint2 c, uint32_t scale) {
  const float s = __uint_as_float(scale << 23);
  auto two = [&](uint32_t w, auto hi) __attribute__((always_inline)) -> uint32_t {
    if constexpr (DT == DT_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, hi.value));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, hi.value));
  };
  constexpr std::false_type lo;
  constexpr std::true_type hi;
  return make_uint4(two(c.x, lo), two(c.x, hi), two(c.y, lo), two(c.y, hi));
}

// A wave takes R8_TOKENS tokens: lane i looks up token i % R8_TOKENS, then the wave passes over
// their pieces of 8 codes, R8_AHEAD of them a lane on their way, so that a store of the wave is 1 KB
// in a piece.  131 K tokens of 8 heads of 128, 619 MB: 121 us, 5.1 TB/s, what a copy reaches (16 codes
// a lane, stores of 16 bytes every 32: 148 us).
constexpr int R8_TOKENS = 8, R8_AHEAD = 8;

template <int DT, int D>
__global__ __launch_bounds__(256) void read8_kernel(Read8Args a) {
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const Ragged& r = a.r;
  const int t0 = (int)min((long long)r.rows, ((long long)blockIdx.x * 4 + wave) * R8_TOKENS), n = min(R8_TOKENS, r.rows - t0);
  if (n <= 0) return;
  // this lane's token: its place in the cache, -1 where it has none, -2 behind the last sequence
  long long place = -2;
  {
    const int t = t0 + min(lane % R8_TOKENS, n - 1), b = seq_of_row(r, t);
    if (b >= 0) {
      const SeqRows s = seq_rows(r, b);
      const int p = t - s.row0, id = p < s.len ? page_id(r, s, p / r.page) : -1;
      place = id < 0 ? -1 : (long long)id * r.page + p % r.page;
    }
  }
  const int per = a.hkv * (D / 8), total = n * per;  // pieces of a token
  int u = lane / per, i = lane % per;
  const int du = kWave / per, di = kWave % per;
  for (int at = lane; at - lane < total; at += kWave * R8_AHEAD) {
    long long from[R8_AHEAD];
    size_t to[R8_AHEAD];
    uint2 kw[R8_AHEAD], vw[R8_AHEAD];
    uint32_t kb[R8_AHEAD], vb[R8_AHEAD];
#pragma unroll
    for (int x = 0; x < R8_AHEAD; x++) {
      const int token = min(u, n - 1);
      from[x] = (long long)(uint32_t)__shfl((int)(uint32_t)place, token) | (long long)__shfl((int)(place >> 32), token) << 32;
      if (at + x * kWave >= total) from[x] = -2;
      to[x] = ((size_t)(t0 + u) * per + i) * 8;
      const size_t row = (size_t)max(from[x], 0ll), head = row * a.hkv + i / (D / 8), piece = (row * per + i) * 8;
      kw[x] = vw[x] = make_uint2(0, 0);
      kb[x] = vb[x] = 0;
      if (from[x] >= 0) {
        const uint64_t k = *(const YR_G uint64_t*)(a.kc + piece);
        const uint64_t v = *(const YR_G uint64_t*)(a.vc + piece);
        kw[x] = make_uint2((uint32_t)k, (uint32_t)(k >> 32));
        vw[x] = make_uint2((uint32_t)v, (uint32_t)(v >> 32));
        kb[x] = gptr(a.ks)[head];
        vb[x] = gptr(a.vs)[head];
      }
      u += du;
      i += di;
      if (i >= per) {
        i -= per;
        u++;
      }
    }
#pragma unroll
    for (int x = 0; x < R8_AHEAD; x++) {
      if (from[x] < -1) continue;
      stg16_stream(a.k + to[x], values8<DT>(kw[x], kb[x]));
      stg16_stream(a.v + to[x], values8<DT>(vw[x], vb[x]));
    }
  }
}

}  // namespace yr

using namespace yr;

extern "C" int yr_hip_append_kv_paged_fp8(const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                                          void* v_cache, void* k_scale, void* v_scale, const void* cos_table,
                                          const void* sin_table, int table_dtype, int max_pos, const void* q_norm,
                                          const void* k_norm, float eps, const int32_t* positions, const int32_t* qo_indptr,
                                          const int32_t* kv_indptr, const int32_t* kv_indices, int n_indices,
                                          const int32_t* kv_len, int rows, int batch, int hq, int hkv, int d, int page_size,
                                          int num_pages, const int64_t* strides7, int dtype, void* stream) {
  const char* nm = "yr_hip_append_kv_paged_fp8";
  Append8Args a;
  a.r = Ragged{qo_indptr, kv_indptr, kv_indices, kv_len, rows, batch, page_size, n_indices, num_pages};
  if (!k || !v || !k_cache || !v_cache || !k_scale || !v_scale || !strides7) return fail(YR_E_INVALID, "%s: null pointer", nm);
  if (!q != !q_out) return fail(YR_E_INVALID, "%s: q and q_out come together", nm);
  if (!cos_table != !sin_table) return fail(YR_E_INVALID, "%s: cos and sin come together", nm);
  if (positions && !cos_table) return fail(YR_E_INVALID, "%s: positions choose rows of the tables: both are needed", nm);
  int rc = ragged_check(nm, a.r, q ? hq : 0, hkv, d, dtype);
  if (rc != YR_OK) return rc;
  if (q && hq <= 0) return fail(YR_E_INVALID, "%s: hq must be positive", nm);
  if (q_norm && !q) return fail(YR_E_INVALID, "%s: q_norm needs q", nm);
  if (cos_table && ((table_dtype != YR_DTYPE_F32 && table_dtype != dtype) || max_pos <= 0))
    return fail(YR_E_INVALID, "%s: tables are fp32 or of k's type, with at least one position", nm);
  const uintptr_t low = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_cache |
                        (uintptr_t)v_cache | (uintptr_t)cos_table | (uintptr_t)sin_table | (uintptr_t)q_norm | (uintptr_t)k_norm;
  if (low & 15) return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  for (int i = q ? 0 : 3; i < 7; i++)
    if (strides7[i] % 8) return fail(YR_E_INVALID, "%s: strides must be multiples of 8 elements", nm);
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.q_out = (uint16_t*)q_out;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.ks = (uint8_t*)k_scale;
  a.vs = (uint8_t*)v_scale;
  a.cos = cos_table;
  a.sin = sin_table;
  a.q_norm = (const uint16_t*)q_norm;
  a.k_norm = (const uint16_t*)k_norm;
  a.positions = positions;
  a.q_row = strides7[0];
  a.q_grp = strides7[1];
  a.q_head = strides7[2];
  a.k_row = strides7[3];
  a.k_head = strides7[4];
  a.v_row = strides7[5];
  a.v_head = strides7[6];
  a.hq = q ? hq : 0;
  a.hkv = hkv;
  a.max_pos = max_pos;
  a.eps = eps;
  if ((long long)a.hq + 2ll * hkv > 1 << 20) return fail(YR_E_INVALID, "%s: too many heads", nm);
  const int per = A8_ROWS * kWave / (d / 16);
  a.chunks = (a.hq + 2 * hkv + per - 1) / per;
  const long long blocks = ((long long)rows * a.chunks + A8_THREADS / kWave - 1) / (A8_THREADS / kWave);
  if (blocks > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
  const bool f32 = table_dtype == YR_DTYPE_F32;
  hipStream_t st = (hipStream_t)stream;
#define YR_A8(DT_, D_, F_)                                                                                     \
  if (dtype == DT_ && d == D_ && f32 == F_)                                                                    \
    hipLaunchKernelGGL((append8_kernel<DT_, D_, F_>), dim3((unsigned)blocks), dim3(A8_THREADS), 0, st, a);
  YR_A8(DT_F16, 64, false) YR_A8(DT_F16, 64, true) YR_A8(DT_F16, 128, false) YR_A8(DT_F16, 128, true)
  YR_A8(DT_BF16, 64, false) YR_A8(DT_BF16, 64, true) YR_A8(DT_BF16, 128, false) YR_A8(DT_BF16, 128, true)
#undef YR_A8
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}

extern "C" int yr_hip_read_kv_paged_fp8(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                                        const int32_t* kv_indptr, const int32_t* kv_indices, int n_indices,
                                        const int32_t* kv_len, const int32_t* out_indptr, void* k_out, void* v_out, int rows,
                                        int batch, int hkv, int d, int page_size, int num_pages, int dtype, void* stream) {
  const char* nm = "yr_hip_read_kv_paged_fp8";
  Read8Args a;
  a.r = Ragged{out_indptr, kv_indptr, kv_indices, kv_len, rows, batch, page_size, n_indices, num_pages};
  if (!k_cache || !v_cache || !k_scale || !v_scale || !out_indptr || !k_out || !v_out)
    return fail(YR_E_INVALID, "%s: null pointer", nm);
  int rc = ragged_check(nm, a.r, 0, hkv, d, dtype);
  if (rc != YR_OK) return rc;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k_out | (uintptr_t)v_out) & 15)
    return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  if (hkv > 1 << 20) return fail(YR_E_INVALID, "%s: too many heads", nm);
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.ks = (const uint8_t*)k_scale;
  a.vs = (const uint8_t*)v_scale;
  a.k = (uint16_t*)k_out;
  a.v = (uint16_t*)v_out;
  a.hkv = hkv;
  const unsigned blocks = (unsigned)(((long long)rows + 4 * R8_TOKENS - 1) / (4 * R8_TOKENS));
  hipStream_t st = (hipStream_t)stream;
#define YR_R8(DT_, D_) \
  if (dtype == DT_ && d == D_) hipLaunchKernelGGL((read8_kernel<DT_, D_>), dim3(blocks), dim3(256), 0, st, a);
  YR_R8(DT_F16, 64) YR_R8(DT_F16, 128) YR_R8(DT_BF16, 64) YR_R8(DT_BF16, 128)
#undef YR_R8
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
