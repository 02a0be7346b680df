// Log probabilities of given tokens, the distribution's entropy and its top
// alternatives, of rows of logits x (f16, bf16 or fp32):
//
//   m = max x, s = sum e^(x - m), logprob = x[token] - m - log s,
//   H = -sum p log p = log s - t / s, t = sum e^(x - m) (x - m),
//   the `top` largest values, equal ones by the lowest index.
//
// One pass over the row.  A wave keeps the running maximum of what it has seen
// (the same in all lanes) and s, t relative to it; both terms of H are then
// non-negative, so nothing cancels, and the largest term of s is exactly 1.
// A row is split over up to 64 workgroups when there are few rows; their
// records are joined by the one that arrives last.
//
// The top costs a few instructions a tile: a lane remembers its largest
// exponent, and the top-th largest of the 64 lanes' is a bound that `top` values
// reach.  Tiles with a lane at or above it are noted and looked at, those lanes
// alone, when the pass is over and the bound of all waves is known.  Keys order by
// value, then by the lower index, so the result does not depend on what else was noted.
//
// NaN values take no part in the top (as in argmax) and make the sums NaN; a
// row of nothing but -inf has no distribution: NaN too.  A token outside
// [0, n_valid) has log probability NaN.
//
// Bound by memory for many rows (2048 of 128256 in bf16, 525 MB, top 5: 97 us, 5.4
// TB/s; without a top 83), by the chain of loads, waves, splits and ranks for few
// (one row 13 us, 64 of 50001 13).
#include <type_traits>

#include "attn_device.h"

namespace yr {

struct LogprobArgs {
  const void* x;
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  float* top_lp;     // [rows][top]
  int64_t* top_ids;  // [rows][top]
  uint64_t* records; // [rows][splits][3 + top]: m, s, t (doubles), keys in order
  uint32_t* tickets; // [rows]
  long long stride;  // elements between rows
  int n, top, splits, chunk;  // chunk: pieces per split
};

constexpr int LP_THREADS = 256;
constexpr int LP_WAVES = LP_THREADS / kWave;
constexpr int LP_MAX_TOP = 64;    // a bound comes from 64 lane maxima
constexpr int LP_BUF = 256;       // candidates a wave holds
constexpr int LP_MAX_SPLITS = 64; // lists that one wave joins, a lane each
constexpr int LP_HITS = 128;      // candidate tiles a wave notes (in the candidates' place)
constexpr int LP_VALUES = 32;     // values per lane and tile (8: 16 rows of 128256 23.5 for 14.6 us, 1 row 11.9 for 12.0)
constexpr int LP_TARGET_WG = 1024; // (512: 256 rows of 32000 16.1 for 15.9 us; 2048: of 128256 34.7 for 26.6)
// |m| beyond which one fma an exponent does not do: c's step is 1/8 here, so m's own exponent
// m log2 e - c is at most 1/16 off 0 and costs no bits; from 2^31 on it may reach 128, where 2^z
// leaves fp32, and near the type's end c itself does.
constexpr float kFar = 0x1p20f;

// A tile with candidates: the lanes that have them, its first piece, its
// largest exponent.
struct LogprobHit {
  uint64_t lanes;
  int p0;
  float high;
};
static_assert(LP_HITS * sizeof(LogprobHit) <= LP_BUF * sizeof(uint64_t), "the list shares the buffer");

constexpr int LP_ITEMS = 512;     // (tile, lane) pairs a workgroup looks at

// Order of a value and its index as one number: larger is better.  0: none.
__device__ __forceinline__ uint64_t lp_key(float v, int i) {
  const uint32_t b = __float_as_uint(v + 0.f);  // -0 ties with 0
  return (uint64_t)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int lp_index(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

template <int C>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, C, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = max(v, dpp_u<0xB1>(v));
  v = max(v, dpp_u<0x4E>(v));
  v = max(v, dpp_u<0x141>(v));
  v = max(v, dpp_u<0x140>(v));
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r[0], r[1]);
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
  const uint32_t hi = wave_max_u((uint32_t)(k >> 32));
  const uint32_t lo = wave_max_u((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ float wave_maxf(float v) {
  v = row16_max(v);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// The larger of three, NaN left out (one instruction).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// (fmaxf(a, b) where a is not a signalling NaN: no instruction to make sure of that)
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// A value that is the same in all lanes, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int l) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}

// A bound that `top` of the 64 lanes' values reach (top <= 64, no NaN), and no
// other lane's where values differ: their order as whole numbers, found bit by bit
// until exactly `top` reach what is set.
__device__ __forceinline__ float lane_bound(float v, int top) {
  if (top == 1) return wave_maxf(v);
  const uint32_t b = __float_as_uint(v), k = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
  uint32_t least = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const int n = __popcll(__ballot(k >= (least | 1u << bit)));
    if (n >= top) least |= 1u << bit;
    if (n == top) break;
  }
  if (least < 0x007fffffu) return -INFINITY;  // (all 64 reach it: numbers before that one are NaN)
  return __uint_as_float(least & 0x80000000u ? least ^ 0x80000000u : ~least);
}

// How many of the 64 lanes' keys beat this lane's.
__device__ __forceinline__ int wave_rank(uint64_t k) {
  int r = 0;
#pragma unroll 8
  for (int l = 0; l < kWave; l++) r += lane_u64(k, l) > k;
  return r;
}

// How many of the n keys at `list` (LDS) beat k; reads run 8 ahead.
__device__ __forceinline__ int rank_in(const uint64_t* list, int n, uint64_t k) {
  int r = 0, j = 0;
  for (; j + 8 <= n; j += 8)
#pragma unroll
    for (int i = 0; i < 8; i++) r += list[j + i] > k;
  for (; j < n; j++) r += list[j] > k;
  return r;
}

// The `top` best of a wave's `count` keys in `buf`, in order, written back to
// buf[0, top) (0 where there are fewer).  Keys differ from one another.
__device__ __forceinline__ void wave_top(uint64_t* buf, int count, int top) {
  const int lane = threadIdx.x % kWave;
  if (count <= kWave && top <= 8) {
    uint64_t k = lane < count ? buf[lane] : 0;
    for (int j = 0; j < top; j++) {
      const uint64_t best = wave_max_key(k);
      if (lane == 0) buf[j] = best;
      if (k == best) k = 0;
    }
  } else if (count <= kWave) {
    const uint64_t k = lane < count ? buf[lane] : 0;
    const int r = wave_rank(k);
    if (lane < top) buf[lane] = 0;
    if (k && r < top) buf[r] = k;
  } else {
    uint64_t k[LP_BUF / kWave];
#pragma unroll
    for (int i = 0; i < LP_BUF / kWave; i++) k[i] = i * kWave + lane < count ? buf[i * kWave + lane] : 0;
    for (int j = 0; j < top; j++) {
      uint64_t b = k[0];
#pragma unroll
      for (int i = 1; i < LP_BUF / kWave; i++) b = k[i] > b ? k[i] : b;
      const uint64_t best = wave_max_key(b);
      if (lane == 0) buf[j] = best;
#pragma unroll
      for (int i = 0; i < LP_BUF / kWave; i++) k[i] = k[i] == best ? 0 : k[i];
    }
  }
}

// The values of a 16-byte piece, and the largest of them (NaN left out).
template <int DT>
__device__ __forceinline__ void unpack_piece(uint4 w, float* v) {
  if constexpr (DT == YR_DTYPE_F32) {
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
  } else {
    v[0] = lo16<DT>(w.x); v[1] = hi16<DT>(w.x); v[2] = lo16<DT>(w.y); v[3] = hi16<DT>(w.y);
    v[4] = lo16<DT>(w.z); v[5] = hi16<DT>(w.z); v[6] = lo16<DT>(w.w); v[7] = hi16<DT>(w.w);
  }
}
template <int DT>
__device__ __forceinline__ float piece_max(uint4 w) {
  constexpr int EPP = DT == YR_DTYPE_F32 ? 4 : 8;
  float v[EPP];
  unpack_piece<DT>(w, v);
  float m = v[0];
#pragma unroll
  for (int e = 1; e < EPP; e++) m = fmaxf(m, v[e]);
  return m;
}

// s = sum 2^z and t = sum 2^z z, z relative to the exponent `from`, brought to `to`.
__device__ __forceinline__ void lp_rescale(double& s, double& t, double from, double to) {
  if (from == to || s == 0) return;  // (NaN stays)
  const double d = from - to, f = __builtin_amdgcn_exp2f((float)d);
  t = f == 0 ? 0 * t : f * (t + d * s);
  s *= f;
}

// The exponent of e^m, exact in 64 bits up to the constant's rounding.
__device__ __forceinline__ double lp_exponent(float m) { return (double)m * (double)kLog2e; }

__device__ __forceinline__ void st_u64(uint64_t* p, uint64_t v) {
  __hip_atomic_store((YR_G uint64_t*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t ld_u64(const uint64_t* p) {
  return __hip_atomic_load((const YR_G uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int DT>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(LogprobArgs a) {
  constexpr int EPP = DT == YR_DTYPE_F32 ? 4 : 8;  // elements per 16-byte piece
  constexpr int U = LP_VALUES / EPP;                       // pieces per lane and tile
  constexpr int ES = 16 / EPP;
  constexpr int kTile = kWave * U, kStep = LP_WAVES * kTile;  // pieces
  __shared__ uint64_t s_buf[LP_WAVES][LP_BUF];
  extern __shared__ uint64_t s_list[];  // [top], then (splits > 1) the splits' candidates
  __shared__ int s_item[LP_ITEMS];  // first pieces of lanes with candidates
  __shared__ int s_items, s_cands;
  __shared__ float s_m[LP_WAVES], s_bound[LP_WAVES];
  __shared__ double s_s[LP_WAVES], s_t[LP_WAVES];
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const char* const x = (const char*)a.x + (size_t)row * a.stride * ES;
  auto at = [&](int i) __attribute__((always_inline)) -> float {
    if constexpr (DT == YR_DTYPE_F32) return gptr((const float*)x)[i];
    else return ld_elem<DT>(gptr((const uint16_t*)x)[i]);
  };
  // the given token's logit, on its way from the start
  float given = NAN;
  if (tid == 0) {
    const int64_t tok = gptr(a.tokens)[row];
    if (tok >= 0 && tok < a.n) given = at((int)tok);
  }

  // Pieces are 16-byte blocks of memory; piece p holds elements p EPP - lead ..
  // and lies inside the row but for the first and the last one.
  const int lead = (int)((uintptr_t)x & 15) / ES;
  const int np = (a.n + lead + EPP - 1) / EPP;
  const int p_begin = split * a.chunk, p_end = min(np, p_begin + a.chunk);
  const int p_first = p_begin + wave * kTile;
  // Piece p; -inf stands for what is not there: it adds nothing and is told
  // apart by its index.
  auto piece = [&](int p) __attribute__((always_inline)) -> uint4 {
    constexpr uint32_t none = DT == DT_F16 ? 0xfc00fc00u : DT == DT_BF16 ? 0xff80ff80u : 0xff800000u;
    const int i0 = p * EPP - lead;
    if (p < p_end && i0 >= 0 && i0 + EPP <= a.n) return ldg16_stream(x - lead * ES + (size_t)p * 16);
    uint64_t f[2] = {(uint64_t)none << 32 | none, (uint64_t)none << 32 | none};
    if (p < p_end) {  // the row's first or last piece
#pragma unroll 1
      for (int e = max(0, -i0); e < min(EPP, a.n - i0); e++) {
        const int sh = 8 * ES * (e % (EPP / 2));
        const uint64_t mask = (((uint64_t)1 << 8 * ES) - 1) << sh;
        uint64_t bits;
        if constexpr (DT == YR_DTYPE_F32) bits = gptr((const uint32_t*)x)[i0 + e];
        else bits = gptr((const uint16_t*)x)[i0 + e];
        if (e < EPP / 2) f[0] = (f[0] & ~mask) | bits << sh;
        else f[1] = (f[1] & ~mask) | bits << sh;
      }
    }
    return make_uint4((uint32_t)f[0], (uint32_t)(f[0] >> 32), (uint32_t)f[1], (uint32_t)(f[1] >> 32));
  };
  // A lane's pieces of tile p0.
  auto load = [&](int p0, uint4* w) __attribute__((always_inline)) {
    if ((p0 > 0 || lead == 0) && (p0 + kTile) * EPP - lead <= a.n && p0 + kTile <= p_end) {
      const char* const tile = x - lead * ES + (size_t)p0 * 16;  // uniform
#pragma unroll
      for (int u = 0; u < U; u++) w[u] = ldg16_stream(tile + (uint32_t)(16 * lane + 16 * kWave * u));
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) w[u] = piece(p0 + u * kWave + lane);
    }
  };

  // ---- sums.  Terms are 2^z, z = x log2 e - c with c = m log2 e rounded: one
  // fma each (m: the largest value so far, -inf: none yet).  s and t are
  // relative to the exponent c and are brought to m log2 e itself at the end.
  // Where m is far off (a mask of -1e9 or the type's lowest value, infinity) z is
  // (x - m) log2 e, exact next to m whatever its size, and they are relative to
  // m log2 e itself.
  float m = -INFINITY, c = 0.f, zm = -INFINITY;  // zm: m's own z
  bool far = false;
  double s = 0, t = 0;
  // Candidates for the top: tiles with a lane whose largest exponent z + c is
  // at least `bound`, the top-th largest of the lanes' maxima.  z + c is off by
  // rounding, by less than `slack` and 2^-18 of itself.
  float high = -INFINITY, bound = -INFINITY, slack = 0.f;
  int hits = 0, fresh = 0;  // entries; how many since the bound moved
  LogprobHit* const hit = reinterpret_cast<LogprobHit*>(s_buf[wave]);
  uint4 next[U];
  if (p_first < p_end) load(p_first, next);
  for (int p0 = p_first; p0 < p_end; p0 += kStep) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; u++) w[u] = next[u];
    if (p0 + kStep < p_end) load(p0 + kStep, next);  // in flight while this tile is worked on
    float z[U][EPP], mz, ex;  // mz: the largest; ex: its value's own exponent
    auto largest = [&]() __attribute__((always_inline)) -> float {
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; u++) mx = fmaxf(mx, piece_max<DT>(w[u]));
      return mx;
    };
    auto exponents = [&]() __attribute__((always_inline)) {
      if (far) {  // (uniform)
#pragma unroll
        for (int u = 0; u < U; u++) {
          unpack_piece<DT>(w[u], z[u]);
#pragma unroll
          for (int e = 0; e < EPP; e++) z[u][e] = (z[u][e] - m) * kLog2e;
        }
        const float mx = largest();
        mz = (mx - m) * kLog2e;
        ex = mx * kLog2e;
        return;
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        unpack_piece<DT>(w[u], z[u]);
#pragma unroll
        for (int e = 0; e < EPP; e++) z[u][e] = fmaf(z[u][e], kLog2e, -c);
      }
      // (of canonical values, unlike the unpacked ones: a maximum is one instruction)
      mz = z[0][0];
#pragma unroll
      for (int j = 1; j + 1 < U * EPP; j += 2) mz = max3(mz, z[j / EPP][j % EPP], z[(j + 1) / EPP][(j + 1) % EPP]);
      mz = max2(mz, z[U - 1][EPP - 1]);
      ex = mz + c;
    };
    bool move = m == -INFINITY;
    if (!move) {
      exponents();
      move = __ballot(mz > zm) != 0;
    }
    if (move) {  // a new maximum, or the first tile
      const float mx = uniform(wave_maxf(largest()));
      if (mx > m) {
        const double was = far ? lp_exponent(m) : (double)c;
        m = mx;
        far = fabsf(m) > kFar;
        c = uniform(m * kLog2e);
        zm = far ? 0.f : uniform(fmaf(m, kLog2e, -c));
        lp_rescale(s, t, was, far ? lp_exponent(m) : (double)c);
        if (!far) slack = fmaxf(slack, 0x1p-18f * fabsf(c));
      }
      exponents();
    }
    float st = 0.f, tt = 0.f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      float es = 0.f;
#pragma unroll
      for (int e = 0; e < EPP; e++) {
        const float p = __builtin_amdgcn_exp2f(z[u][e]);
        es += p;
        tt = fmaf(p, max2(z[u][e], -1e4f), tt);  // (0 * -inf is none)
      }
      st += es;
    }
    s += st;
    t += tt;
    if (a.top > 0) {
      high = max2(high, ex);
      const uint64_t lanes = __ballot(!(ex < bound - slack));
      if (lanes) {
        if (hits == LP_HITS) {  // drop what the bound has passed
          int kept = 0;
          for (int i = 0; i < hits; i++) {
            const LogprobHit h = hit[i];
            if (!(h.high < bound - slack)) hit[kept++] = h;
          }
          hits = kept < LP_HITS ? kept : LP_HITS + 1;  // too many: every tile is a candidate
        }
        if (hits < LP_HITS) {
          const float th = uniform(wave_maxf(ex));
          hit[hits++] = LogprobHit{lanes, p0, th};
        }
        if (++fresh > 2 || bound == -INFINITY) {
          fresh = 0;
          const float b = uniform(lane_bound(high, a.top));
          const float lower = b - 0x1p-17f * fabsf(b) - slack;  // below what b stands for
          if (lower > bound && lower < INFINITY) bound = lower;
        }
      }
    }
  }
  if (!far && m > -INFINITY) lp_rescale(s, t, c, lp_exponent(m));
  s = wave_sum_d(s);
  t = wave_sum_d(t);
  if (lane == 0) {
    s_m[wave] = m;
    s_s[wave] = s;
    s_t[wave] = t;
    s_bound[wave] = bound;
  }
  if (tid == 0) s_items = s_cands = 0;
  for (int i = tid; i < a.top; i += LP_THREADS) s_list[i] = 0;
  __syncthreads();

  // ---- the top.  What the lanes with candidates hold, at or above the bound of
  // all waves, goes to one list of keys, and a key's place is the number that beat it.
  if (a.top > 0) {
#pragma unroll
    for (int w = 0; w < LP_WAVES; w++) bound = fmaxf(bound, s_bound[w]);
    bound = uniform(bound);
    // the same bound for a value: x log2 e >= bound
    const float b = bound * 0.693147180559945309f;
    const float xb = bound > -INFINITY ? b - 0x1p-18f * fabsf(b) : -INFINITY;
    const float least = bound - slack;
    const uint64_t live = __ballot(!(high < least));
    for (int j = 0; j < min(hits, LP_HITS); j++) {
      const LogprobHit h = hit[j];
      const uint64_t lanes = uniform(h.lanes) & live;
      if (h.high < least || !lanes) continue;
      int base = 0;
      if (lane == 0) base = atomicAdd(&s_items, __popcll(lanes));
      base = __builtin_amdgcn_readfirstlane(base) + __popcll(lanes & ((1ull << lane) - 1));
      if (((lanes >> lane) & 1) && base < LP_ITEMS) s_item[base] = h.p0 + lane;
    }
    if (hits > LP_HITS && lane == 0) atomicAdd(&s_items, LP_ITEMS + 1);
    __syncthreads();
    const int items = s_items;
    uint64_t* const cand = s_buf[0];
    constexpr int kCands = LP_WAVES * LP_BUF;
    if (items <= LP_ITEMS) {
      for (int i = tid; i < items * U; i += LP_THREADS) {
        const int p = s_item[i / U] + i % U * kWave;
        float v[EPP];
        unpack_piece<DT>(piece(p), v);
#pragma unroll
        for (int e = 0; e < EPP; e++) {
          const int at = p * EPP - lead + e;
          if (v[e] >= xb && p < p_end && at >= 0 && at < a.n) {
            const int c = atomicAdd(&s_cands, 1);
            if (c < kCands) cand[c] = lp_key(v[e], at);
          }
        }
      }
      __syncthreads();
    }
    const int cands = s_cands;
    if (items <= LP_ITEMS && cands <= kCands) {
      for (int i = tid; i < cands; i += LP_THREADS) {
        const uint64_t k = cand[i];
        const int r = rank_in(cand, cands, k);
        if (r < a.top) s_list[r] = k;
      }
    } else {
      // Too many: equal values in their thousands, as in a row that a mask has
      // left nearly empty.  Each wave goes over its pieces once more, keeping
      // its best keys; those above `worst` are still wanted.
      uint64_t* const buf = s_buf[wave];
      uint64_t worst = 0;
      int count = 0;
      __syncthreads();
      for (int p0 = p_first; p0 < p_end; p0 += kStep)
#pragma unroll 1
        for (int u = 0; u < U; u++) {
          const int i0 = (p0 + u * kWave + lane) * EPP - lead;
          float v[EPP];
          unpack_piece<DT>(piece(p0 + u * kWave + lane), v);
#pragma unroll 1
          for (int e = 0; e < EPP; e++) {
            const float f = v[0];
#pragma unroll
            for (int i = 0; i + 1 < EPP; i++) v[i] = v[i + 1];
            const int at = i0 + e;
            const uint64_t k = f >= xb && p0 + u * kWave + lane < p_end && at >= 0 && at < a.n ? lp_key(f, at) : 0;
            if (count + kWave > LP_BUF) {
              wave_top(buf, count, a.top);
              count = a.top;  // (the buffer was fuller than top)
              worst = uniform(buf[a.top - 1]);
            }
            const uint64_t take = __ballot(k > worst);
            if (k > worst) buf[count + __popcll(take & ((1ull << lane) - 1))] = k;
            count += __popcll(take);
          }
        }
      wave_top(buf, count, a.top);
      __syncthreads();
      for (int i = tid; i < LP_WAVES * a.top; i += LP_THREADS) {
        const uint64_t k = s_buf[i / a.top][i % a.top];
        int r = 0;
#pragma unroll
        for (int w = 0; w < LP_WAVES; w++) r += rank_in(s_buf[w], a.top, k);
        if (k && r < a.top) s_list[r] = k;
      }
    }
  }
  __syncthreads();
  // ---- the waves' numbers
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < LP_WAVES; w++) M = fmaxf(M, s_m[w]);
  s = t = 0;
#pragma unroll
  for (int w = 0; w < LP_WAVES; w++) {
    double sw = s_s[w], tw = s_t[w];
    lp_rescale(sw, tw, lp_exponent(s_m[w]), lp_exponent(M));
    s += sw;
    t += tw;
  }
  __syncthreads();

  if (a.splits > 1) {
    const int rec_len = 3 + a.top;
    uint64_t* rec = a.records + (size_t)row * a.splits * rec_len;
    if (tid == 0) {
      st_u64(rec + (size_t)split * rec_len, (uint64_t)__double_as_longlong(lp_exponent(M)));
      st_u64(rec + (size_t)split * rec_len + 1, (uint64_t)__double_as_longlong(s));
      st_u64(rec + (size_t)split * rec_len + 2, (uint64_t)__double_as_longlong(t));
    }
    for (int i = tid; i < a.top; i += LP_THREADS) st_u64(rec + (size_t)split * rec_len + 3 + i, s_list[i]);
    if (!arrive_last(&a.tickets[row], a.splits)) return;
    // The splits' ordered lists.  Where `some` of them have their deep-th key at or
    // above a bound, deep * some >= top keys are: what is below the bound is out,
    // and the few others are ranked.
    const int keys = a.splits * a.top, deep = (a.top + a.splits - 1) / a.splits;
    const int some = deep ? (a.top + deep - 1) / deep : 0;
    uint64_t* const cand = s_list + a.top;  // (room for every key)
    const bool listed = tid < a.splits;
    double ms = -INFINITY, ss = 0, ts = 0;
    uint64_t head = 0;
    if (listed) {
      const uint64_t* const r = rec + (size_t)tid * rec_len;
      ms = __longlong_as_double((long long)ld_u64(r));
      ss = __longlong_as_double((long long)ld_u64(r + 1));
      ts = __longlong_as_double((long long)ld_u64(r + 2));
      if (a.top > 0) head = ld_u64(r + 2 + deep);
    }
    constexpr int KU = 8;  // keys of a thread in flight
    uint64_t got[KU];
    auto fetch = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < KU; u++) {
        const int i = i0 + u * LP_THREADS;
        got[u] = i < keys ? ld_u64(rec + (size_t)(i / a.top) * rec_len + 3 + i % a.top) : 0;
      }
    };
    fetch(tid);
    if (wave == 0) {
      // (a float times the constant: the division gives the float back)
      M = wave_maxf((float)(ms / (double)kLog2e));
      lp_rescale(ss, ts, ms, lp_exponent(M));
      s = wave_sum_d(ss);
      t = wave_sum_d(ts);
      if (a.top > 0) {
        const float b = lane_bound(head ? lp_value(head) : -INFINITY, some);
        if (lane == 0) {
          s_cands = 0;
          s_bound[0] = b;
        }
      }
    }
    for (int i = tid; i < a.top; i += LP_THREADS) s_list[i] = 0;
    __syncthreads();
    if (a.top > 0) {
      const float b = s_bound[0];
      for (int i = tid;;) {
#pragma unroll
        for (int u = 0; u < KU; u++)
          if (got[u] && lp_value(got[u]) >= b) cand[atomicAdd(&s_cands, 1)] = got[u];
        i += KU * LP_THREADS;
        if (i >= keys) break;
        fetch(i);
      }
      __syncthreads();
      const int cands = s_cands;
      for (int i = tid; i < cands; i += LP_THREADS) {
        const uint64_t k = cand[i];
        const int r = rank_in(cand, cands, k);
        if (r < a.top) s_list[r] = k;
      }
      __syncthreads();
    }
    if (wave != 0) return;
  }
  if (M == -INFINITY) s = t = NAN;  // no value at all
  if (s < 1) s = 1;                 // the largest term alone, but for its rounding
  const double ls = log(s);
  if (tid == 0) {
    gptr(a.logprob)[row] = (float)((double)(given - M) - ls);
    gptr(a.entropy)[row] = (float)(ls - t / s * 0.693147180559945309);
  }
  if (tid < a.top) {
    const uint64_t k = s_list[tid];
    gptr(a.top_lp)[(size_t)row * a.top + tid] = k ? (float)((double)(lp_value(k) - M) - ls) : -INFINITY;
    gptr(a.top_ids)[(size_t)row * a.top + tid] = k ? lp_index(k) : -1;
  }
}

// A row is split while LP_TARGET_WG workgroups or fewer run, each with one tile of
// all its waves at least (1000 rows of 128256 whole 60 us, in two 64).
struct LogprobPlan {
  int splits, chunk;
};
static LogprobPlan logprobs_plan(int rows, int n, int dtype) {
  const int epp = dtype == YR_DTYPE_F32 ? 4 : 8;
  const int np = (n - 1) / epp + 2;  // pieces; a row off its boundary has one more
  LogprobPlan p;
  const int tile = LP_THREADS * LP_VALUES / epp, most = (np + tile - 1) / tile;
  int sp = LP_TARGET_WG / rows;
  if (sp > LP_MAX_SPLITS) sp = LP_MAX_SPLITS;
  if (sp > most) sp = most;
  if (sp < 1) sp = 1;
  p.chunk = ((np + sp - 1) / sp + tile - 1) / tile * tile;
  p.splits = (np + p.chunk - 1) / p.chunk;
  return p;
}

}  // namespace yr

using namespace yr;

extern "C" size_t yr_hip_token_logprobs_workspace(int rows, int n_valid, int top_n, int dtype) {
  if (rows <= 0 || n_valid <= 0 || top_n < 0) return 0;
  const LogprobPlan p = logprobs_plan(rows, n_valid, dtype);
  return p.splits > 1 ? kTicketBytes + (size_t)rows * p.splits * (3 + top_n) * sizeof(uint64_t) : 0;
}

extern "C" int yr_hip_token_logprobs(const void* x, const int64_t* tokens, float* logprob, float* entropy,
                                     float* top_logprob, int64_t* top_ids, int rows, int n, int n_valid,
                                     int64_t row_stride, int top_n, int dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* nm = "yr_hip_token_logprobs";
  if (!x || !tokens || !logprob || !entropy || (top_n > 0 && (!top_logprob || !top_ids)))
    return fail(YR_E_INVALID, "%s: null pointer", nm);
  if (rows <= 0 || n <= 0 || n_valid <= 0 || n_valid > n || row_stride < n) return fail(YR_E_INVALID, "%s: bad shape", nm);
  if (n > (1 << 30)) return fail(YR_E_INVALID, "%s: %d columns are too many", nm, n);
  if (top_n < 0 || top_n > LP_MAX_TOP || top_n > n_valid)
    return fail(YR_E_INVALID, "%s: top_n %d (at most %d and the valid columns)", nm, top_n, LP_MAX_TOP);
  if (dtype != YR_DTYPE_F16 && dtype != YR_DTYPE_BF16 && dtype != YR_DTYPE_F32)
    return fail(YR_E_INVALID, "%s: dtype", nm);
  const int size = dtype == YR_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)x % size) return fail(YR_E_INVALID, "%s: logits must be aligned to their type", nm);
  const LogprobPlan p = logprobs_plan(rows, n_valid, dtype);
  LogprobArgs a{x,       tokens,     logprob, entropy, top_logprob, top_ids, nullptr,
                nullptr, row_stride, n_valid, top_n,   p.splits,    p.chunk};
  const size_t need = yr_hip_token_logprobs_workspace(rows, n_valid, top_n, dtype);
  if (need > workspace_bytes || (need && !workspace))
    return fail(YR_E_WORKSPACE, "%s: workspace %zu < %zu", nm, workspace_bytes, need);
  if ((long long)rows * a.splits > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
  a.tickets = (uint32_t*)workspace;
  a.records = need ? (uint64_t*)((char*)workspace + kTicketBytes) : nullptr;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * a.splits));
  const size_t lds = (size_t)(a.splits > 1 ? a.splits + 1 : 1) * top_n * sizeof(uint64_t);
#define YR_LP(DT_) \
  if (dtype == DT_) hipLaunchKernelGGL((logprobs_kernel<DT_>), grid, dim3(LP_THREADS), lds, st, a);
  YR_LP(YR_DTYPE_F16) YR_LP(YR_DTYPE_BF16) YR_LP(YR_DTYPE_F32)
#undef YR_LP
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
