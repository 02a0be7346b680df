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

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct SelectArgs {
  Ragged r;
  const uint16_t* q;
  const uint16_t* bounds;  // [pages][hkv][2][D]
  int32_t* out;            // [rows][hkv][top]
  uint64_t* keys;          // [rows][hkv][max_pages] where a row is split
  uint32_t* tickets;       // [rows][hkv]
  int hq, hkv, max_pages, top, first, last, splits, chunk, tile;  // tile: rows
};

constexpr int SEL_MAX_PAGES = 16384;  // 64-bit keys of one row in LDS: 128 of 160 KiB
constexpr int SEL_ROWS = 16;          // rows of a tile
constexpr int SEL_TILE_WAVES = 16;    // a row's list each: 512 rows of 512 pages 21 us, 23 with 8
constexpr int SEL_TILE_PAGES = 4096;  // a tile's keys in LDS: as much, 4 rows at least
constexpr int SEL_MIN_CHUNK = 128;    // pages per split at least

// Whole-number order of a score: larger is better, -0 equals 0, NaN is last.
__device__ __forceinline__ uint64_t score_key(double s) {
  if (s != s) return 0;
  const int64_t b = __double_as_longlong(s + 0.0);
  return b < 0 ? ~(uint64_t)b : (uint64_t)b | 0x8000000000000000ull;
}

template <int C>
__device__ __forceinline__ uint32_t dpp_word(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, C, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_or(uint32_t v) {
  v |= dpp_word<0xB1>(v);
  v |= dpp_word<0x4E>(v);
  v |= dpp_word<0x141>(v);
  v |= dpp_word<0x140>(v);
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = r[0] | r[1];
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return r[0] | r[1];
}
template <int C>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  const uint64_t o = (uint64_t)dpp_word<C>((uint32_t)(b >> 32)) << 32 | dpp_word<C>((uint32_t)b);
  return v + __longlong_as_double((long long)o);
}
// Sum over groups of 16 (8) lanes, every lane the same.
template <int N>
__device__ __forceinline__ double group_sum(double v) {
  v = dpp_add<0x4E>(dpp_add<0xB1>(v));
  v = dpp_add<0x141>(v);
  return N == 16 ? dpp_add<0x140>(v) : v;
}

// Writes the ascending list of a row: pages [0, f) and [n - l, n) and the `m`
// best keys of [f, n - l), -1 behind.  W waves work together (the whole
// workgroup, or one wave by itself); the keys are in LDS, and a lane holds those
// of pages (i W + wave) 64 + lane, i < R, in registers (R = 0: more than 16; they
// are read again each time).
//
// The m-th best key is found bit by bit: of the bits in which the keys differ,
// from the highest, a bit is set when m keys at least reach the value with it.
// That ends as soon as exactly m do, after about log2 n bits.  Several waves take
// two bits a step, which costs three counts and saves an exchange.
template <int W, int R>
__device__ __forceinline__ void choose_from(const uint64_t* key, int n, int f, int l, int m, int top, int32_t* out) {
  __shared__ uint64_t s_cnt[2][W], s_diff[W];
  __shared__ int s_pos[kWave];
  const int lane = threadIdx.x % kWave, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c0 = f, c1 = n - l;  // candidates
  const int turns = R ? R : (n + W * kWave - 1) / (W * kWave);
  uint64_t k[R ? R : 1];
  // key i of this lane; 0 (never counted below) where there is no candidate
  auto get = [&](int i) __attribute__((always_inline)) -> uint64_t {
    if constexpr (R > 0) return k[i];
    const int u = (i * W + wave) * kWave + lane;
    return u >= c0 && u < c1 ? key[u] : 0;
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int u = (i * W + wave) * kWave + lane;
      k[i] = u >= c0 && u < c1 ? key[u] : 0;
    }
  }
  int turn = 0;
  // sums over the waves of three counts of up to 2^21, one barrier for all
  auto all = [&](uint64_t c) __attribute__((always_inline)) -> uint64_t {
    if constexpr (W == 1) return c;
    if (lane == 0) s_cnt[turn][wave] = c;
    __syncthreads();
    uint64_t sum = 0;
#pragma unroll
    for (int w = 0; w < W; w++) sum += s_cnt[turn][w];
    turn ^= 1;  // the next count goes elsewhere: one barrier each
    return sum;
  };
  // how many keys reach a value > 0, or each of three
  auto count = [&](uint64_t least) __attribute__((always_inline)) -> int {
    int c = 0;
#pragma unroll(R ? R : 4)
    for (int i = 0; i < turns; i++) c += __popcll(__ballot(get(i) >= least));
    return (int)all(c);
  };
  auto count3 = [&](uint64_t x, uint64_t y, uint64_t z) __attribute__((always_inline)) -> uint64_t {
    int cx = 0, cy = 0, cz = 0;
#pragma unroll(R ? R : 4)
    for (int i = 0; i < turns; i++) {
      const uint64_t v = get(i);
      cx += __popcll(__ballot(v >= x));
      cy += __popcll(__ballot(v >= y));
      cz += __popcll(__ballot(v >= z));
    }
    return all((uint64_t)cx | (uint64_t)cy << 21 | (uint64_t)cz << 42);
  };
  uint64_t bound = 0;      // keys from it on are taken ..
  int equal = 0x7fffffff;  // .. of those equal to it only the first `equal`
  if (m > 0 && m < c1 - c0) {
    const uint64_t any = key[c0];
    uint64_t diff = 0;
#pragma unroll(R ? R : 4)
    for (int i = 0; i < turns; i++) {
      const int u = (i * W + wave) * kWave + lane;
      if (u >= c0 && u < c1) diff |= get(i) ^ any;
    }
    diff = (uint64_t)wave_or((uint32_t)(diff >> 32)) << 32 | wave_or((uint32_t)diff);
    if constexpr (W > 1) {
      if (lane == 0) s_diff[wave] = diff;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; w++) diff |= s_diff[w];
    }
    int bit = diff ? 63 - __builtin_clzll(diff) : -1;
    bound = bit < 0 ? any : bit == 63 ? 0 : any & ~((2ull << bit) - 1);
    bool exact = false;
    if constexpr (W == 1) {
      for (; bit >= 0 && !exact; bit--) {
        const uint64_t cand = bound | 1ull << bit;
        const int c = count(cand);
        if (c >= m) bound = cand;
        exact = c == m;
      }
    }
    bit |= 1;  // pairs of bits: one above the differing ones comes out as all keys have it
    for (bit--; W > 1 && bit >= 0 && !exact; bit -= 2) {
      const uint64_t step = 1ull << bit, low = bound & ~(3 * step);
      const uint64_t c = count3(low | step, low | 2 * step, low | 3 * step);
      const int c1s = (int)(c & 0x1fffff), c2s = (int)(c >> 21 & 0x1fffff), c3s = (int)(c >> 42);
      const int best = c3s >= m ? 3 : c2s >= m ? 2 : c1s >= m ? 1 : 0;
      bound = low | best * step;
      exact = (best == 3 ? c3s : best == 2 ? c2s : best == 1 ? c1s : -1) == m;
    }
    if (!exact) {  // equal keys at the border: the first of them
      equal = m - (bound == ~0ull ? 0 : count(bound + 1));
    }
  }
  // ascending list; the waves take blocks of 64 pages in turn
  if constexpr (W > 1 && R > 0 && R * W <= kWave) {
    if (equal == 0x7fffffff) {  // (uniform) no ties: one exchange of every block's count
      uint64_t taken[R];
      int mine = 0;  // lane i: block i's
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int u = (i * W + wave) * kWave + lane;
        taken[i] = __ballot(u < n && (u < c0 || u >= c1 || (m > 0 && k[i] >= bound)));
        mine = lane == i ? __popcll(taken[i]) : mine;
      }
      if (lane < R) s_pos[lane * W + wave] = mine;
      __syncthreads();
      int sum = lane < R * W ? s_pos[lane] : 0;  // up to and with block `lane`
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int v = __shfl_up(sum, o);
        if (lane >= o) sum += v;
      }
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int j = i * W + wave, base = j ? __builtin_amdgcn_readlane(sum, j - 1) : 0;
        const int pos = base + __popcll(taken[i] & ((1ull << lane) - 1));
        if ((taken[i] >> lane & 1) && pos < top) gptr(out)[pos] = j * kWave + lane;
      }
      const int all_taken = __builtin_amdgcn_readlane(sum, kWave - 1);
      for (int i = all_taken + (int)threadIdx.x; i < top; i += W * kWave) gptr(out)[i] = -1;
      return;
    }
  }
  int at = 0, eq = 0;  // written so far, keys equal to bound seen so far
#pragma unroll(R ? R : 1)
  for (int i = 0; i < turns; i++) {
    const int u = (i * W + wave) * kWave + lane;
    const bool cand = u >= c0 && u < c1;
    const uint64_t key_u = get(i);
    const bool same = cand && key_u == bound;
    int before = eq;
    const uint64_t be = __ballot(same);
    if (equal != 0x7fffffff) {  // (uniform)
      const int alle = (int)all(__popcll(be));
      if constexpr (W > 1) {
#pragma unroll
        for (int w = 0; w < W; w++)
          if (w < wave) before += (int)s_cnt[turn ^ 1][w];
      }
      eq += alle;
      before += __popcll(be & ((1ull << lane) - 1));
    }
    const bool take = u < n && (!cand || (m > 0 && (same ? before < equal : key_u > bound)));
    const uint64_t bt = __ballot(take);
    int pos = at;
    at += (int)all(__popcll(bt));
    if constexpr (W > 1) {
#pragma unroll
      for (int w = 0; w < W; w++)
        if (w < wave) pos += (int)s_cnt[turn ^ 1][w];
    }
    pos += __popcll(bt & ((1ull << lane) - 1));
    if (take && pos < top) gptr(out)[pos] = u;
  }
  for (int i = at + wave * kWave + lane; i < top; i += W * kWave) gptr(out)[i] = -1;
}

template <int W>
__device__ __forceinline__ void choose(const uint64_t* key, int n, int f, int l, int m, int top, int32_t* out) {
  const int turns = (n + W * kWave - 1) / (W * kWave);
  if (turns <= 1) choose_from<W, 1>(key, n, f, l, m, top, out);
  else if (turns <= 4) choose_from<W, 4>(key, n, f, l, m, top, out);
  else if (turns <= 8) choose_from<W, 8>(key, n, f, l, m, top, out);
  else if (turns <= 16) choose_from<W, 16>(key, n, f, l, m, top, out);
  else choose_from<W, 0>(key, n, f, l, m, top, out);
}

// Pages of a row: visible and existing ones n, forced ones at the start (f) and
// the end (l), and how many of the others are chosen (m).
struct RowPages {
  int n, f, l, m;
};
__device__ __forceinline__ RowPages row_pages(const SelectArgs& a, const SeqRows& s, int p) {
  RowPages r;
  r.n = p < 0 ? 0 : min(min(p / a.r.page + 1, s.npg), a.max_pages);
  r.f = min(a.first, r.n);
  r.l = min(a.last, r.n - r.f);
  r.m = min(max(a.top - r.f - r.l, 0), r.n - r.f - r.l);
  return r;
}

__device__ __forceinline__ void sel_store(uint64_t* p, uint64_t v) {
  __hip_atomic_store((YR_G uint64_t*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t sel_load(const uint64_t* p) {
  return __hip_atomic_load((const YR_G uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A lane's part of a page's score: 8 channels.
template <int DT>
__device__ __forceinline__ double page_dot(const double* down, const double* up, uint4 mn, uint4 mx) {
  const uint32_t w0[4] = {mn.x, mn.y, mn.z, mn.w}, w1[4] = {mx.x, mx.y, mx.z, mx.w};
  double s0 = 0, s1 = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    s0 = fma(down[2 * e], (double)lo16<DT>(w0[e]), s0);
    s1 = fma(up[2 * e], (double)lo16<DT>(w1[e]), s1);
    s0 = fma(down[2 * e + 1], (double)hi16<DT>(w0[e]), s0);
    s1 = fma(up[2 * e + 1], (double)hi16<DT>(w1[e]), s1);
  }
  return s0 + s1;
}

// One row and kv head, its pages split over `splits` workgroups; the last one
// to arrive chooses.  Bound by memory where there are rows enough (32 of 1024 pages,
// 8 kv heads of 128, 105 MB: 27 us, of which the scores 20), else by the chain of
// page id, bounds, tickets, keys and steps of the border (one of 2048 pages 13 us).
template <int DT, int D, int W>
__global__ __launch_bounds__(W * kWave) void select_kernel(SelectArgs a) {
  constexpr int T = W * kWave;
  constexpr int LPP = D / 8, PPB = T / LPP, U = 4;  // lanes per page, pages per pass, passes in flight
  extern __shared__ uint64_t s_key[];
  __shared__ double s_q[2][D];
  const int split = blockIdx.x % a.splits, pair = blockIdx.x / a.splits;
  const int h = pair % a.hkv, t = pair / a.hkv, tid = threadIdx.x;
  const int b = seq_of_row(a.r, t);
  if (b < 0) return;
  const SeqRows s = seq_rows(a.r, b);
  int32_t* out = a.out + (size_t)pair * a.top;
  const RowPages r = row_pages(a, s, s.len - s.n + (t - s.row0));
  const bool scored = r.m > 0 && r.m < r.n - r.f - r.l;
  if (scored) {
    const int g = a.hq / a.hkv;
    for (int d = tid; d < D; d += T) {
      double up = 0, down = 0;
      const uint16_t* q = a.q + ((size_t)t * a.hq + (size_t)h * g) * D + d;
      for (int i0 = 0; i0 < g; i0 += 4) {  // 4 loads in flight
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = gptr(q)[(size_t)min(i0 + i, g - 1) * D];
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (i0 + i < g) {
            const double x = ld_elem<DT>(w[i]);
            up += x > 0 ? x : x != x ? x : 0;
            down += x < 0 ? x : 0;
          }
      }
      s_q[0][d] = down;
      s_q[1][d] = up;
    }
    __syncthreads();
    const int j = tid % LPP;
    double qd[8], qu[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qd[i] = s_q[0][8 * j + i];
      qu[i] = s_q[1][8 * j + i];
    }
    const int begin = max(split * a.chunk, r.f), end = min((split + 1) * a.chunk, r.n - r.l);
    for (int u0 = begin; u0 < end; u0 += U * PPB) {
      int id[U];
      uint4 mn[U], mx[U];
#pragma unroll
      for (int i = 0; i < U; i++) {
        const int u = u0 + i * PPB + tid / LPP;
        id[i] = u < end ? page_id(a.r, s, u) : -1;
      }
#pragma unroll
      for (int i = 0; i < U; i++) {
        // (a page that is not there reads page 0, unused)
        const uint16_t* bd = a.bounds + ((size_t)max(id[i], 0) * a.hkv + h) * 2 * D + 8 * j;
        mn[i] = ldg16(bd);
        mx[i] = ldg16(bd + D);
      }
#pragma unroll
      for (int i = 0; i < U; i++) {
        const double sum = group_sum<LPP>(page_dot<DT>(qd, qu, mn[i], mx[i]));
        const int u = u0 + i * PPB + tid / LPP;
        if (j == 0 && u < end) {
          const uint64_t k = id[i] < 0 ? 0 : score_key(sum);
          if (a.splits > 1) sel_store(a.keys + (size_t)pair * a.max_pages + u, k);
          else s_key[u] = k;
        }
      }
    }
    if (a.splits > 1) {
      if (!arrive_last(&a.tickets[pair], a.splits)) return;
      const uint64_t* const keys = a.keys + (size_t)pair * a.max_pages;
      for (int u0 = r.f + tid; u0 < r.n - r.l; u0 += 8 * T) {  // 8 loads in flight
        uint64_t k[8];
#pragma unroll
        for (int i = 0; i < 8; i++) k[i] = sel_load(keys + min(u0 + i * T, r.n - r.l - 1));
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (u0 + i * T < r.n - r.l) s_key[u0 + i * T] = k[i];
      }
    }
    __syncthreads();
  } else if (split > 0) {
    return;  // nothing to compare: the first workgroup writes the list
  }
  choose<W>(s_key, r.n, r.f, r.l, r.m, a.top, out);
}

// Memory that a wave's lanes wrote, before they read each other's.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// Order of an fp32 score; 0 stands for none.
__device__ __forceinline__ uint32_t rough_key(float s) {
  const uint32_t b = __float_as_uint(s);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float rough_score(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
template <int C>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, dpp_word<C>(v));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(v))));
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r[0], r[1]);
}

// Exact scores by one wave: D / 8 lanes a page, 8 channels each.
template <int DT, int D>
struct ExactRow {
  static constexpr int LPP = D / 8, PP = kWave / LPP;  // lanes per page, pages per pass
  double down[8], up[8];
  // row t, kv head h
  __device__ __forceinline__ void load(const SelectArgs& a, int t, int h) {
    const int g = a.hq / a.hkv;
    const uint16_t* q = a.q + ((size_t)t * a.hq + (size_t)h * g) * D + 8 * (threadIdx.x % LPP);
#pragma unroll
    for (int e = 0; e < 8; e++) down[e] = up[e] = 0;
#pragma unroll 4
    for (int i = 0; i < g; i++) {
      const uint4 v = ldg16(q + (size_t)i * D);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const double x = e % 2 ? hi16<DT>(w[e / 2]) : lo16<DT>(w[e / 2]);
        up[e] += x > 0 ? x : x != x ? x : 0;
        down[e] += x < 0 ? x : 0;
      }
    }
  }
  // keys of the pages page(0) .. page(n - 1) -> out[i]
  template <class F>
  __device__ __forceinline__ void keys(const SelectArgs& a, const SeqRows& s, int h, int n, F page, uint64_t* out) {
    const int lane = threadIdx.x % kWave, j = lane % LPP;
    for (int i0 = 0; i0 < n; i0 += PP) {
      const int i = i0 + lane / LPP, id = i < n ? page_id(a.r, s, page(i)) : -1;
      const uint16_t* bd = a.bounds + ((size_t)max(id, 0) * a.hkv + h) * 2 * D + 8 * j;
      const double sum = group_sum<LPP>(page_dot<DT>(down, up, ldg16(bd), ldg16(bd + D)));
      if (j == 0 && i < n) out[i] = id < 0 ? 0 : score_key(sum);
    }
  }
};

// A wave's border among a row's scores: get(i), i < turns, gives a lane's keys
// (0: none), page(i) the pages they belong to, in order.  With A the m-th best
// score, a page more than 2 err above A is in and one more than 2 err below it is
// out.  Between, where there is a choice, the pages are scored exactly and their
// keys in `key` (LDS) become the verdict, for the caller to read again.  Returns
// the key from which on pages are in; 0: more than 64 of them are too close.
template <int DT, int D, int R, class Get, class Page>
__device__ __forceinline__ uint32_t rough_border(const SelectArgs& a, const SeqRows& s, int m, int t, int h, float err,
                                                 int turns, uint32_t any, Get get, Page page, uint32_t* key, int* list,
                                                 uint64_t* exact, bool* settled) {
  const int lane = threadIdx.x % kWave;
  uint32_t diff = 0;
#pragma unroll(R ? R : 4)
  for (int i = 0; i < turns; i++) diff |= get(i) ? get(i) ^ any : 0;
  diff = wave_or(diff);
  int bit = diff ? 31 - __builtin_clz(diff) : -1;
  uint32_t bound = bit < 0 ? any : bit == 31 ? 0 : any & ~((2u << bit) - 1);
  for (bool split = false; bit >= 0 && !split; bit--) {
    const uint32_t cand = bound | 1u << bit;
    int c = 0;
#pragma unroll(R ? R : 4)
    for (int i = 0; i < turns; i++) c += __popcll(__ballot(get(i) >= cand));
    if (c >= m) bound = cand;
    split = c == m;
  }
  // the worst of those at `bound` or above, which is A, and the best below it
  uint32_t least = 0, next = 0;
  int reach = 0;
#pragma unroll(R ? R : 4)
  for (int i = 0; i < turns; i++) {
    const uint32_t v = get(i);
    reach += __popcll(__ballot(v >= bound));
    least = max(least, v >= bound ? ~v : 0);
    next = max(next, v < bound ? v : 0);
  }
  bound = ~wave_max(least);
  next = wave_max(next);
  const float A = rough_score(bound), low = A - 2 * err, high = A + 2 * err;
  if (reach == m && !(next && rough_score(next) >= low)) return bound;
  *settled = true;
  int n = 0, in = 0;
#pragma unroll(R ? R : 4)
  for (int i = 0; i < turns; i++) {
    const uint32_t k = get(i);
    const float v = rough_score(k);
    const bool sure = k && v > high, band = k && v >= low && !sure;
    const uint64_t b = __ballot(band);
    in += __popcll(__ballot(sure));
    const int at = n + __popcll(b & ((1ull << lane) - 1));
    if (band && at < kWave) list[at] = page(i);
    n += __popcll(b);
  }
  if (n > kWave) return 0;
  wave_sync();
  ExactRow<DT, D> row;
  row.load(a, t, h);
  row.keys(a, s, h, n, [&](int i) { return list[i]; }, exact);
  wave_sync();
  if (lane < n) {
    const uint64_t mine = exact[lane];
    int rank = 0;
    for (int i = 0; i < n; i++) rank += exact[i] > mine || (exact[i] == mine && i < lane);
    key[list[lane]] = rank < m - in ? ~0u : 1u;  // (1: below every score)
  }
  wave_sync();
  return bound;
}

// The list of a row whose scores' keys at `key` (LDS, written over) are within err
// of the exact ones, by one wave; R of the keys a lane in registers (0: read
// again).  False: too many are too close.
template <int DT, int D, int R>
__device__ __forceinline__ bool choose_rough(const SelectArgs& a, const SeqRows& s, const RowPages& r, int t, int h, float err,
                                             uint32_t* key, int* list, uint64_t* exact, int32_t* out) {
  const int lane = threadIdx.x % kWave, c0 = r.f, c1 = r.n - r.l;
  const int turns = R ? R : (r.n + kWave - 1) / kWave;
  uint32_t k[R ? R : 1];
  auto read = [&](int i) __attribute__((always_inline)) -> uint32_t {
    const int u = i * kWave + lane;
    return u >= c0 && u < c1 ? key[u] : 0;
  };
  auto get = [&](int i) __attribute__((always_inline)) -> uint32_t {
    if constexpr (R > 0) return k[i];
    return read(i);
  };
  auto keep = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < R; i++) k[i] = read(i);
  };
  keep();
  uint32_t bound = 0;
  if (r.m > 0 && r.m < c1 - c0) {
    if (r.m <= kWave) {
      // The m-th best of the lanes' best keys bounds A from below, and few pages
      // are above it: up to 64 of them go to a list, and the rest is done there.
      uint32_t best = 0, least = 0;
#pragma unroll(R ? R : 4)
      for (int i = 0; i < turns; i++) best = max(best, get(i));
      if (c1 - c0 > kWave)  // (fewer: all of them)
        for (int bit = 31; bit >= 0; bit--) {
          const int c = __popcll(__ballot(best >= (least | 1u << bit)));
          if (c >= r.m) least |= 1u << bit;
          if (c == r.m) break;
        }
      const float from = rough_score(least) - 2.125f * err;
      int n = 0;
#pragma unroll(R ? R : 4)
      for (int i = 0; i < turns; i++) {
        const uint32_t v = get(i);
        const bool near = v && !(rough_score(v) < from);  // (least may stand for NaN: all of them)
        const uint64_t b = __ballot(near);
        const int at = n + __popcll(b & ((1ull << lane) - 1));
        if (near && at < kWave) list[at] = i * kWave + lane;
        n += __popcll(b);
      }
      if (n <= kWave) {
        wave_sync();
        const int mine = lane < n ? list[lane] : 0;
        uint32_t v = lane < n ? key[mine] : 0;
        wave_sync();
        bool settled = false;
        bound = rough_border<DT, D, 1>(a, s, r.m, t, h, err, 1, __builtin_amdgcn_readfirstlane(v),
                                       [&](int) { return v; }, [&](int) { return mine; }, key, list, exact, &settled);
        if (settled) v = lane < n ? key[mine] : 0;
        const uint64_t b = __ballot(v >= bound && lane < n);
        const int taken = __popcll(b);  // m
        if (b >> lane & 1) gptr(out)[r.f + __popcll(b & ((1ull << lane) - 1))] = mine;
        for (int i = lane; i < a.top - taken; i += kWave) {
          const int j = i < r.f ? i : i + taken;
          gptr(out)[j] = i < r.f ? i : i - r.f < r.l ? c1 + i - r.f : -1;
        }
        return true;
      }
    }
    bool settled = false;
    bound = rough_border<DT, D, R>(a, s, r.m, t, h, err, turns, key[c0], get, [&](int i) { return i * kWave + lane; }, key,
                                   list, exact, &settled);
    if (bound == 0) return false;
    if (settled) keep();
  }
  int at = 0;
#pragma unroll(R ? R : 4)
  for (int i = 0; i < turns; i++) {
    const int u = i * kWave + lane;
    const bool take = u < r.n && (u < c0 || u >= c1 || (r.m > 0 && get(i) >= bound));
    const uint64_t b = __ballot(take);
    const int pos = at + __popcll(b & ((1ull << lane) - 1));
    if (take && pos < a.top) gptr(out)[pos] = u;
    at += __popcll(b);
  }
  for (int i = at + lane; i < a.top; i += kWave) gptr(out)[i] = -1;
  return true;
}

// Up to 16 rows of one sequence and one kv head.  Their scores are a product of
// [16][2 D] by [2 D][pages] on the 16-bit matrix instruction: Q- and Q+ (fp32) as
// the sum of three bf16 parts, or of two f16 parts after a scaling by row, against
// the bounds as they come from memory.  (In fp32 on 16x16x4 the loop takes 15
// instead of 10 us at 512 rows of 512 pages, on the 64-bit one 24.)
//
// The list is that of the exact scores all the same: products of the parts are
// exact, and a score's error is at most that of adding up D products in each of two
// sums, a step of fp32 each (half of one if the instruction rounds to nearest), of
// Q's own g terms, of the parts' rest and of joining the sums, all relative to
// sum |Q| |bound| <= |Q| |bound| (Euclidean norms, the largest of any page).  Pages
// nearer to the border than that allows are scored in 64 bits, as are all of a row
// with numbers too large, too small or not finite.
//
// 512 rows of 512 pages, 8 kv heads of 128: 22 us, of which Q 3, the scores 10, a
// row's list for each wave 5; with keys 100 of their spread off zero 27, where every
// score has to be exact (all alike, infinite) 120 to 170.
template <int DT, int D>
__global__ __launch_bounds__(SEL_TILE_WAVES * kWave) void select_tile_kernel(SelectArgs a) {
  constexpr int C = D / 32;                   // 16-byte pieces per lane of each bound
  constexpr int L = DT == DT_F16 ? 2 : 3;     // parts of Q
  constexpr float kPart = DT == DT_F16 ? 2048.f : 1.f;
  constexpr int QS = 2 * D + 8;               // a row of Q- and Q+ (padded: rows start in other banks)
  extern __shared__ uint64_t s_key[];         // [tile][stride], fp32 keys in the first half of each row's
  __shared__ int s_tile[2];
  __shared__ uint32_t s_odd, s_norm;          // rows that need 64 bits throughout, the largest squared norm of a page
  __shared__ float s_q2[SEL_ROWS], s_scale[SEL_ROWS];  // squared norms of Q, what its parts were divided by
  struct Lists {
    uint64_t exact[kWave];
    int list[kWave];
  };
  __shared__ union __attribute__((aligned(16))) {
    uint16_t q[L][SEL_ROWS][QS];
    Lists w[SEL_TILE_WAVES];  // after the scores
  } s_u;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int h = blockIdx.x % a.hkv, tile = blockIdx.x / a.hkv, stride = a.max_pages;
  if (tid == 0) {
    find_tile(a.r, tile, a.tile, s_tile);
    s_odd = s_norm = 0;
  }
  __syncthreads();
  const int b = __builtin_amdgcn_readfirstlane(s_tile[0]), i0 = __builtin_amdgcn_readfirstlane(s_tile[1]);
  if (b >= a.r.batch) return;
  const SeqRows s = seq_rows(a.r, b);
  const int nt = min(a.tile, s.n - i0), t0 = s.row0 + i0, p0 = s.len - s.n + i0;
  const RowPages last = row_pages(a, s, p0 + nt - 1);  // the row that sees most
  const int g = a.hq / a.hkv, col = lane % 16, grp = lane / 16;
  if (last.m > 0 && last.m < last.n - last.f - last.l) {
    // Q and its parts, 4 channels of each sign a thread, a row in D / 4 lanes of a wave
    for (int i = tid; i < SEL_ROWS * (D / 4); i += SEL_TILE_WAVES * kWave) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      const uint16_t* q = a.q + ((size_t)(t0 + min(row, nt - 1)) * a.hq + (size_t)h * g) * D + d;
      float x[8] = {};  // Q-, Q+
#pragma unroll 4
      for (int j = 0; j < g; j++) {
        const u32x2 v = *(const YR_G u32x2*)(q + (size_t)j * D);
        const float y[4] = {lo16<DT>(v.x), hi16<DT>(v.x), lo16<DT>(v.y), hi16<DT>(v.y)};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[4 + e] += y[e] > 0 ? y[e] : y[e] != y[e] ? y[e] : 0;
          x[e] += y[e] < 0 ? y[e] : 0;
        }
      }
      float q2 = 0, most = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        q2 = fmaf(x[e], x[e], q2);
        most = fmaxf(most, fabsf(x[e]));
      }
#pragma unroll
      for (int o = 1; o < D / 4; o <<= 1) {
        q2 += __shfl_xor(q2, o);
        most = fmaxf(most, __shfl_xor(most, o));
      }
      // f16 parts of numbers up to 2^15
      const int up = DT == DT_F16 && most > 0 && most < INFINITY ? 15 - (ilogbf(most) + 1) : 0;
      if (d == 0) {
        s_q2[row] = q2;
        s_scale[row] = ldexpf(1.f, -up);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = ldexpf(x[e], up);
#pragma unroll
      for (int part = 0; part < L; part++)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const u32x2 w = {pack2<DT>(x[e], x[e + 1]), pack2<DT>(x[e + 2], x[e + 3])};
          *(u32x2*)&s_u.q[part][row][(e ? D : 0) + d] = w;
          const float y[4] = {lo16<DT>(w.x), hi16<DT>(w.x), lo16<DT>(w.y), hi16<DT>(w.y)};
#pragma unroll
          for (int j = 0; j < 4; j++) x[e + j] = (x[e + j] - y[j]) * kPart;
        }
    }
    __syncthreads();
    float scale[4];
#pragma unroll
    for (int i = 0; i < 4; i++) scale[i] = s_scale[4 * grp + i];
    float norm = 0;
    uint32_t odd = 0;
    // 16 pages a turn and wave; the next turn's bounds are on their way
    auto fetch = [&](int u0, uint4* v) __attribute__((always_inline)) -> int {
      const int u = u0 + col, id = u < last.n ? page_id(a.r, s, u) : -1;
      const uint16_t* bd = a.bounds + ((size_t)max(id, 0) * a.hkv + h) * 2 * D + 8 * grp;
#pragma unroll
      for (int c = 0; c < 2 * C; c++) v[c] = ldg16(bd + c / C * D + c % C * 32);
      return id;
    };
    uint4 next[2 * C];
    int id_next = fetch(16 * wave, next);
    for (int u0 = 16 * wave; u0 < last.n; u0 += 16 * SEL_TILE_WAVES) {
      uint4 v[2 * C];
#pragma unroll
      for (int c = 0; c < 2 * C; c++) v[c] = next[c];
      const int u = u0 + col, id = id_next;
      if (u0 + 16 * SEL_TILE_WAVES < last.n) id_next = fetch(u0 + 16 * SEL_TILE_WAVES, next);
      f32x4 acc[L][2] = {};
      float b2 = 0;
      int row = col;  // (hidden: 96 registers of Q would not fit, so it is read from LDS each turn)
      asm volatile("" : "+v"(row));
#pragma unroll
      for (int c = 0; c < 2 * C; c++) {
#pragma unroll
        for (int part = 0; part < L; part++) {
          const uint4 q = *(const uint4*)&s_u.q[part][row][c / C * D + c % C * 32 + 8 * grp];
          acc[part][c / C] = mfma16<DT>(q, v[c], acc[part][c / C]);
        }
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          b2 = fmaf(lo16<DT>(w[e]), lo16<DT>(w[e]), b2);
          b2 = fmaf(hi16<DT>(w[e]), hi16<DT>(w[e]), b2);
        }
      }
      b2 += __shfl_xor(b2, 16);
      b2 += __shfl_xor(b2, 32);
      if (u < last.n) {
        norm = fmaxf(norm, b2);
        if (id < 0 || !(b2 < INFINITY)) odd = 0xffff;
        // result rows 4 grp + i, page col
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float sum = acc[L - 1][0][i] + acc[L - 1][1][i];
#pragma unroll
          for (int part = L - 2; part >= 0; part--) sum = fmaf(sum, 1.f / kPart, acc[part][0][i] + acc[part][1][i]);
          sum *= scale[i];
          if (!(fabsf(sum) < INFINITY)) odd |= 1u << (4 * grp + i);
          if (4 * grp + i < nt) reinterpret_cast<uint32_t*>(s_key + (size_t)(4 * grp + i) * stride)[u] = rough_key(sum);
        }
      }
    }
    if (odd) atomicOr(&s_odd, odd);
    norm = __uint_as_float(wave_max(__float_as_uint(norm)));
    if (lane == 0) atomicMax(&s_norm, __float_as_uint(norm));
  }
  __syncthreads();
  for (int i = wave; i < nt; i += SEL_TILE_WAVES) {
    const RowPages r = row_pages(a, s, p0 + i);
    int32_t* const out = a.out + ((size_t)(t0 + i) * a.hkv + h) * a.top;
    uint64_t* const key = s_key + (size_t)i * stride;
    const bool scored = r.m > 0 && r.m < r.n - r.f - r.l;
    const float b2 = __uint_as_float(s_norm), q2 = s_q2[i];
    bool done = !scored;
    if (!scored || (!(s_odd >> i & 1) && b2 > 1e-30f && b2 < 1e30f && q2 > 1e-30f && q2 < 1e30f)) {
      const float err = scored ? (float)(D + 8 + g) * (0x1p-23f * (1.f + 1.f / 32)) * (sqrtf(b2) * sqrtf(q2)) : 0.f;
      uint32_t* const rough = reinterpret_cast<uint32_t*>(key);
      int* const list = s_u.w[wave].list;
      uint64_t* const exact = s_u.w[wave].exact;
      const int turns = (r.n + kWave - 1) / kWave;
      done = turns <= 4    ? choose_rough<DT, D, 4>(a, s, r, t0 + i, h, err, rough, list, exact, out)
             : turns <= 8  ? choose_rough<DT, D, 8>(a, s, r, t0 + i, h, err, rough, list, exact, out)
             : turns <= 16 ? choose_rough<DT, D, 16>(a, s, r, t0 + i, h, err, rough, list, exact, out)
                           : choose_rough<DT, D, 0>(a, s, r, t0 + i, h, err, rough, list, exact, out);
    }
    if (!done) {
      ExactRow<DT, D> row;
      row.load(a, t0 + i, h);
      row.keys(a, s, h, r.n, [](int i) { return i; }, key);
      wave_sync();
      choose_from<1, 0>(key, r.n, r.f, r.l, r.m, a.top, out);
    }
  }
}

}  // namespace yr

using namespace yr;

// Rows of a tile: as many as have room for their keys.
static int select_tile_rows(int max_pages) {
  int tile = SEL_ROWS;
  while (tile > 1 && tile * max_pages > SEL_MAX_PAGES) tile /= 2;
  return tile;
}

// Rows of the same sequence share their pages' bounds in a tile, but a tile is one
// workgroup's work, and a row by itself spreads over the chip.  As measured (8 kv
// heads of 128) tiles take 10 us and 1 us for 57 pages, once per 256 of them, and
// rows 8 us and 1 us for 19400 pages of all rows and heads.  Tiles and rows, us: one
// sequence of 1024 pages, 16 rows 30 and 22, 32 rows 28 and 23, 48 rows 28 and 35; 512
// rows of 512 pages 21 and 98, of 2048 93 and 333; 8 rows of 8 sequences, 512 pages,
// 18 and 20; 16 of 4, 128 pages, 12.4 and 10.1; 4 of 64, 128 pages, 30 and 19.
static bool select_tiled(bool ragged, long long tiles, long long pairs, int hkv, int max_pages) {
  if (!ragged || max_pages > SEL_TILE_PAGES) return false;
  const long long rounds = (tiles * hkv + 255) / 256;
  return rounds * (570 + max_pages) < 456 + pairs * max_pages / 340;
}

// Rows per tile of a call and its tiles at most, whatever the sequences' rows; 0: row by row.
static int select_tile_plan(bool ragged, int rows, int batch, int hkv, int max_pages, long long* tiles) {
  const int tile = select_tile_rows(max_pages);
  *tiles = (long long)rows / tile + batch;
  if (*tiles > rows) *tiles = rows;
  return select_tiled(ragged, *tiles, (long long)rows * hkv, hkv, max_pages) ? tile : 0;
}

// Waves per workgroup and splits per row: as many as run at once, 16 waves a CU (one
// split more, 24 rows of 1024 pages: 38.3 us for 24.4).  Times with 8 kv heads of 128:
//   16 waves where every row and head then has a workgroup for itself at once, and
//   for rows whose keys would not fit into the registers of 8: 18 rows of 1024 pages
//   23.8 (8 waves 25.0), 32 of 256 13.1 (15.2), 32 of 1024 26.9 (32.6), 4 of 6144 36.2
//   (42.4), 8 of 8192 56 (64); but 1 of 2048 17.4 (13.2), 40 of 1024 43.1 (38.2);
//   4 waves for more rows than 8 of them run at once, and for few pages: 64 rows of
//   64 pages 8.3 (8 waves 10.1), 128 of 64 10.4 (17.5), 256 of 128 27.6 (37.4), 128
//   of 512 41.7 (44.3); but 64 of 256 19.8 (17.1).
struct SelectPlan {
  int waves, splits, chunk;
};
static SelectPlan select_plan(long long pairs, int max_pages) {
  SelectPlan p;
  p.waves = max_pages >= 6144                 ? 16
            : max_pages <= 64 || pairs > 512  ? 4
            : pairs > 128 && pairs <= 256     ? 16
                                              : 8;
  const long long target = 256 * 16 / p.waves;
  long long sp = target > pairs ? target / pairs : 1;
  const int most = (max_pages + SEL_MIN_CHUNK - 1) / SEL_MIN_CHUNK;
  if (sp > most) sp = most;
  p.chunk = (int)((max_pages + sp - 1) / sp);
  p.splits = (max_pages + p.chunk - 1) / p.chunk;
  return p;
}

extern "C" size_t yr_hip_select_pages_workspace(int rows, int hkv, int page_size, int max_kv_len) {
  if (rows <= 0 || hkv <= 0 || page_size <= 0 || max_kv_len <= 0) return 0;
  const long long pairs = (long long)rows * hkv;
  const int max_pages = (max_kv_len - 1) / page_size + 1;
  return select_plan(pairs, max_pages).splits > 1 ? kTicketBytes + (size_t)pairs * max_pages * sizeof(uint64_t) : 0;
}

extern "C" int yr_hip_select_pages_plan(int rows, int batch, int ragged, int hkv, int page_size, int max_kv_len, int* plan3) {
  const char* nm = "yr_hip_select_pages_plan";
  if (!plan3 || rows <= 0 || batch <= 0 || hkv <= 0 || page_size <= 0 || max_kv_len <= 0 ||
      (max_kv_len - 1) / page_size >= SEL_MAX_PAGES)
    return fail(YR_E_INVALID, "%s: shape", nm);
  const int max_pages = (max_kv_len - 1) / page_size + 1;
  const SelectPlan p = select_plan((long long)rows * hkv, max_pages);
  long long tiles;
  plan3[0] = select_tile_plan(ragged != 0, rows, batch, hkv, max_pages, &tiles);
  plan3[1] = plan3[0] ? SEL_TILE_WAVES : p.waves;
  plan3[2] = plan3[0] ? 1 : p.splits;
  return YR_OK;
}

// A launch with `lds` bytes of dynamic LDS.
template <class K>
static int select_launch(const char* nm, K kernel, unsigned grid, int threads, size_t lds, hipStream_t st, const SelectArgs& a) {
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return check_hip(e, nm);
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), lds, st, a);
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}

extern "C" int yr_hip_select_pages(const void* q, const void* page_bounds, const int32_t* qo_indptr,
                                   const int32_t* kv_indptr, const int32_t* kv_indices, int n_indices,
                                   const int32_t* kv_len, int32_t* pages, int rows, int batch, int hq, int hkv, int d,
                                   int page_size, int num_pages, int max_kv_len, int top_pages, int first_pages,
                                   int last_pages, int dtype, void* workspace, size_t workspace_bytes,
                                   void* stream) {
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
  const SelectPlan p = select_plan((long long)rows * hkv, a.max_pages);
  a.splits = p.splits;
  a.chunk = p.chunk;
  const size_t need = yr_hip_select_pages_workspace(rows, hkv, page_size, max_kv_len);
  if (need > workspace_bytes || (need && !workspace))
    return fail(YR_E_WORKSPACE, "%s: workspace %zu < %zu", nm, workspace_bytes, need);
  a.tickets = (uint32_t*)workspace;
  a.keys = need ? (uint64_t*)((char*)workspace + kTicketBytes) : nullptr;
  long long tiles;
  a.tile = select_tile_plan(qo_indptr != nullptr, rows, batch, hkv, a.max_pages, &tiles);
  const bool tiled = a.tile > 0;
  const size_t lds = (size_t)a.max_pages * 8 * (tiled ? a.tile : 1);
  const unsigned grid = (unsigned)(tiled ? tiles * hkv : (long long)rows * hkv * a.splits);
  hipStream_t st = (hipStream_t)stream;
#define YR_SEL(DT_, D_)                                                                        \
  if (dtype == DT_ && d == D_)                                                                 \
    return tiled ? select_launch(nm, select_tile_kernel<DT_, D_>, grid, SEL_TILE_WAVES * kWave, lds, st, a) \
           : p.waves == 4 ? select_launch(nm, select_kernel<DT_, D_, 4>, grid, 4 * kWave, lds, st, a)      \
           : p.waves == 8 ? select_launch(nm, select_kernel<DT_, D_, 8>, grid, 8 * kWave, lds, st, a)      \
                          : select_launch(nm, select_kernel<DT_, D_, 16>, grid, 16 * kWave, lds, st, a);
  YR_SEL(DT_F16, 64) YR_SEL(DT_F16, 128) YR_SEL(DT_BF16, 64) YR_SEL(DT_BF16, 128)
#undef YR_SEL
  return fail(YR_E_INVALID, "%s: shape", nm);
}
