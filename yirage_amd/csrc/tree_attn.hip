// GQA attention of new rows (single tokens, trees of drafted tokens, chunks of prompts)
// over a paged cache in 16 bits or in e4m3 with a power of two per token and head.
//
//   out[t] = sum_j p_j v_j / sum_j p_j,  p_j = exp(q_t k_j / sqrt(D))
//
// over the tokens before the sequence's new ones, and of the new ones those at or before
// row t's place, or those that tree_mask[t] names.
//
// A tile is consecutive rows of one sequence with their G heads: 16, 32, 64 or 128 columns of
// the products, which are transposed (S^T = K Q^T and O^T += V^T P^T on MFMA 16x16x32; a
// lane holds one query row of each 16).  Up to 32 columns every wave holds all of them and the
// waves split the tokens; wider tiles share each block of tokens, 16 or 32 columns a wave (16
// sequences' trees of 16 nodes and 4 heads, 64 columns: 69 us, as private tiles of 32 columns 93).
// One pass with a running maximum; statistics and O are fp32.  The weights are rounded to q's type
// before they meet V (half a step of a weight each; their sum takes them unrounded).
//
// In 8 bits a fragment is converted between LDS and MFMA.  The conversion multiplies by
// a power of two, so a key is read with its scale for nothing and without rounding (down to
// bf16's smallest normal number); a fragment of V holds 8 tokens, whose scales go into the
// weights' exponents instead.
//
// Bound: single rows by memory (32 sequences of 4 to 8 K tokens in 8 bits, 436 MB, 84 us, 5.2 TB/s; in 16 bits
// 865 MB, 152 us, 5.7 TB/s), one long row by the chain of ids, first block, merge and join (32 K tokens: 20 + 4 us);
// chunks by issue and the waits between MFMA and softmax of two waves a SIMD (2048 rows after 14 K tokens in 8 bits,
// 503 GFLOP, 599 us, 0.84 PFLOP/s: VALU 65 % and MFMA 36 % of a SIMD's cycles).  Of the two workgroups of a CU the
// one that starts first runs some 10 % faster; larger shares for those: the chunk 620 -> 607, a prompt of 2048
// 90 -> 100, so not kept.
#include <type_traits>

#include "attn_device.h"
#include "ragged.h"

namespace yr {

// The figures of these choices are replayed calls of 32 / 8 heads of 128, a graph's launch included.
constexpr int TR_WAVES = 4;
// Workgroups: one a CU where each has loads enough of its own on their way (one row over 32 K tokens
// 32.6 us, with 512 of them 35.7, 320: 39.2; 32 rows of d = 64 65, 70 and 85), two where waves wait for
// a shared block (64-node trees 144 us, with 256 194, 1024: 160; a chunk of 2048 641, 1083, 659).
constexpr int TR_PRIVATE_WG = 256, TR_SHARED_WG = 512;
// From that many tiles (of all kv heads) on each has a workgroup: 500 sequences of 1000 tokens 170 us, in equal
// parts 195, 200 trees of 8 nodes 118 and 142; 160 sequences of 2000 tokens are cut, 122 us for 128 (300 of
// 1500: 175 us, in equal parts 162).  All of these of one length.  The rule asks for no length, and a sequence much
// longer than the rest is then one workgroup's: 256 single rows, one over 32 K tokens and the others over 1 K,
// take 1000 us, 255 of them, which are cut, 125.
constexpr int TR_MANY = 2048;
constexpr int TR_MIN_BLOCKS = 4;   // of a part: one row over 8 K tokens 24.6 us, with 2 26.9, with 8 25.5
// Of a tile's start, in tokens, at its front (spread over its tokens: 64-node trees 144 us for 132, a prompt of
// 2048 104 for 95, without 153): 16 trees of 15 nodes 56 us, with 128 59, with 320 62.
constexpr int TR_TILE_COST = 192;
constexpr int TR_SHORT = 512;      // tiles of so many tokens on average are not split: 7 trees over 57 tokens 18 us for 35
constexpr int TR_WAVE_BLOCKS = 8;  // of a wave, for several heads to share a workgroup: 32 rows of d = 64 70 us, never 94; with 2 one row 37.3 for 35.7
// Fragments that are read from LDS ahead of their products (left to the compiler each was waited for:
// a chunk of 2048 rows over 16 bits 620 us for 568, 64-node trees 132 for 123; 1 ahead 577 and 124, 4: 563 and 126).
constexpr int TR_FRAGMENTS = 2;
// Tokens of a block: a lane's each, half as many where a wave has a block of its own and a
// token 256 bytes (shared ones of 32: a chunk of 2048 rows in 16 bits 744 us for 629).
constexpr int tr_block(int row_bytes, bool share) { return row_bytes == 256 && !share ? 32 : 64; }

struct TreeArgs {
  Ragged r;
  const uint16_t* q;    // [rows][hq][D]
  const uint8_t* kc;    // [pages][page][hkv][D], 16 or 8 bits
  const uint8_t* vc;
  const uint8_t* ks;    // [pages][page][hkv] (8 bits)
  const uint8_t* vs;
  const uint8_t* mask;  // [rows][mask_cols], rows mask_row apart, or null
  uint16_t* out;
  float* partial;       // [hkv][parts heads][2][tt G][D + 4]: O, m, l
  int4* split;          // .x the parts of this call; then [hkv][parts heads]: first row, columns and parts (0: none)
                        // of the tile that begins in a part and ends in another
  long long mask_row;
  int mask_cols, hq, hkv, tt;  // rows per tile
  int parts, log_heads;        // workgroups per kv head (0: one a tile); kv heads that may share one
  uint32_t page_mul, page_shift;       // x / page = x page_mul >> page_shift for x < 2^31
  float scale_log2, scale_inv;
};

// Work.  A sequence of n new rows has ceil(n / tt) tiles, and a tile counts for as many units
// as tokens its last row may see, and TR_TILE_COST for its start.  The units of a kv head, one
// sequence after another, are cut into `parts` equal ranges, a workgroup each (below TR_MANY tiles): lengths
// that differ leave no workgroup waiting, a long sequence is split and several short ones share a workgroup.
// (Each tile split as often as the longest needs: 64-node trees over 16 bits 169 us for 145, one
// row over 32 K tokens 29 for 25.)  The cut is made on the device, from lengths that no host reads.
struct SeqWork {
  SeqRows s;
  int tiles;
  long long units;
};
__device__ __forceinline__ long long units_before(const TreeArgs& a, const SeqRows& s, int tile) {
  if (a.mask) return (long long)tile * (s.len + TR_TILE_COST);
  return (long long)tile * (max(s.len - s.n, 0) + TR_TILE_COST) + (long long)a.tt * tile * (tile + 1) / 2;
}
__device__ __forceinline__ SeqWork seq_work(const TreeArgs& a, int b) {
  SeqWork w;
  w.tiles = 0;
  w.units = 0;
  if (b < a.r.batch) {
    w.s = seq_rows(a.r, b);
    w.tiles = (w.s.n + a.tt - 1) / a.tt;
    w.units = units_before(a, w.s, w.tiles);
  }
  return w;
}
__device__ __forceinline__ long long lane64(long long x, int lane) {  // (uniform lane)
  return (long long)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane) |
         (long long)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32;
}
__device__ __forceinline__ long long first64(long long x) { return lane64(x, 0); }
// sum over the lanes up to this one, in registers
template <int CTRL, int ROWS>
__device__ __forceinline__ long long dpp_add64(long long x) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return x + ((long long)(uint32_t)lo | (long long)hi << 32);
}
__device__ __forceinline__ long long scan64(long long x) {
  x = dpp_add64<0x111, 0xf>(x);  // rows of 16 lanes: 1, 2, 4, 8 to the right
  x = dpp_add64<0x112, 0xf>(x);
  x = dpp_add64<0x114, 0xf>(x);
  x = dpp_add64<0x118, 0xf>(x);
  x = dpp_add64<0x142, 0xa>(x);  // lane 15 of rows 0 and 2 to the rows behind them
  return dpp_add64<0x143, 0xc>(x);  // lane 31 to the upper half
}
// Units and tiles of a kv head.  Each wave for itself, a sequence a lane; w: the first 64 sequences.
__device__ __forceinline__ long long all_units(const TreeArgs& a, const SeqWork& w, long long* tiles) {
  long long sum = w.units, count = w.tiles;
  for (int b = kWave; b < a.r.batch; b += kWave) {
    const SeqWork more = seq_work(a, b + (int)threadIdx.x % kWave);
    sum += more.units;
    count += more.tiles;
  }
  *tiles = lane64(scan64(count), kWave - 1);
  return lane64(scan64(sum), kWave - 1);
}
// A tile: its sequence (batch: none), number in it, first unit and units.
struct TileAt {
  SeqRows s;
  int b, tile;
  long long from, units;
};
__device__ __forceinline__ SeqRows seq_of_lane(const SeqRows& s, int lane) {  // (uniform lane)
  return SeqRows{__builtin_amdgcn_readlane(s.row0, lane), __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.len, lane),
                 __builtin_amdgcn_readlane(s.pg0, lane), __builtin_amdgcn_readlane(s.npg, lane)};
}
// The one that unit x falls into.
__device__ __forceinline__ TileAt find_unit(const TreeArgs& a, SeqWork w, long long x) {
  TileAt t;
  t.b = a.r.batch;
  long long before = 0;
  for (int b = 0; b < a.r.batch; b += kWave) {
    if (b > 0) w = seq_work(a, b + (int)threadIdx.x % kWave);
    const long long sum = scan64(w.units);
    const uint64_t past = __ballot(before + sum > x);
    if (past) {
      const int i = __builtin_ctzll(past);
      t.b = b + i;
      t.s = seq_of_lane(w.s, i);
      before += lane64(sum - w.units, i);
      // the last tile that begins at or before x
      int lo = 0, hi = __builtin_amdgcn_readlane(w.tiles, i);
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (before + units_before(a, t.s, mid) <= x) lo = mid;
        else hi = mid;
      }
      t.tile = lo;
      t.from = before + units_before(a, t.s, lo);
      t.units = before + units_before(a, t.s, lo + 1) - t.from;
      return t;
    }
    before += lane64(sum, kWave - 1);
  }
  return t;
}
// Tile `index` of all (a workgroup each, where there are many more than run at once).
__device__ __forceinline__ TileAt find_index(const TreeArgs& a, SeqWork w, int index) {
  TileAt t;
  t.b = a.r.batch;
  t.tile = 0;
  t.from = 0;
  t.units = 1;
  if (!a.r.qo_indptr) {
    // (a call made for more parts than it has sequences: those behind the last have no tables to read)
    if (index < a.r.batch) {
      t.b = index;
      t.s = seq_rows(a.r, index);
    }
    return t;
  }
  long long left = index;
  for (int b = 0; b < a.r.batch; b += kWave) {
    if (b > 0) w = seq_work(a, b + (int)threadIdx.x % kWave);
    const long long sum = scan64(w.tiles);
    const uint64_t past = __ballot(sum > left);
    if (past) {
      const int i = __builtin_ctzll(past);
      t.b = b + i;
      t.s = seq_of_lane(w.s, i);
      t.tile = (int)(left - lane64(sum - w.tiles, i));
      return t;
    }
    left -= lane64(sum, kWave - 1);
  }
  return t;
}

// The units behind the first tile's start (every part has one such start) are cut into `parts` ranges
// that differ by one at most: where range w begins, and the one that holds unit u.  (In fp64 instead
// of 64-bit divisions the kernel needs more registers: 64-node trees 155 us for 131.)
__device__ __forceinline__ long long part_start(long long units, int parts, int w) {
  const long long cut = max(units - TR_TILE_COST, 0ll);
  return w == 0 ? 0 : TR_TILE_COST + cut / parts * w + min((long long)w, cut % parts);
}
__device__ __forceinline__ int part_of(long long units, int parts, long long u) {
  const long long cut = max(units - TR_TILE_COST, 0ll), per = cut / parts, more = cut % parts, longer = (per + 1) * more;
  const long long at = max(u - TR_TILE_COST, 0ll);
  return __builtin_amdgcn_readfirstlane((int)(at < longer ? at / (per + 1) : more + (at - longer) / max(per, 1ll)));
}
// 8 consecutive e4m3 codes of LDS rows, transposed across each 16-lane group: lanes 2 e
// and 2 e + 1 address the halves of row e's 16 bytes, lane i receives byte i of rows 0 .. 7.
typedef int v2i32 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i32 lds_v2i32;
__device__ __forceinline__ uint2 lds_tr8(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i32*)p));
}

// 4 codes times 2^n (given as a float) -> 4 values of 16 bits
template <int DT>
__device__ __forceinline__ uint2 e4m3x4(uint32_t w, float s) {
  if constexpr (DT == DT_BF16)
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true)));
  else
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true)));
}

// 16-byte chunk permutations of an LDS row of RB bytes.  K fragments read one chunk
// column of 16 consecutive rows, V fragments a chunk (8 bits) or half a chunk pair
// (16 bits) of 4 or 2 x 4 rows: any 8 lanes of either hit 8 chunks apart modulo 128 bytes.
template <int RB>
__device__ __forceinline__ int tk_swz(int row) {
  return RB == 256 ? row & 15 : RB == 128 ? row & 7 : (row >> 1) & 3;
}
template <bool Q8, int RB>
__device__ __forceinline__ int tv_swz(int row) {
  if constexpr (Q8) return RB == 128 ? (row & 3) | ((row >> 4) & 1) << 2 : ((row >> 1) & 1) | ((row >> 4) & 1) << 1;
  else return RB == 256 ? ((row & 7) << 1) | ((row >> 3) & 1) : (row & 3) << 1;
}

// Bytes j .. j + 3 of a row of n, 0 for those outside of it.  (One load of 4 bytes inside the
// row, whatever its alignment.)
__device__ __forceinline__ uint32_t mask4(const uint8_t* row, int n, int j) {
  if (n >= 4) {
    const int at = min(max(j, 0), n - 4), off = j - at;
    uint32_t w;
    __builtin_memcpy(&w, (const YR_G uint8_t*)gptr(row) + at, 4);
    return off <= -4 || off >= 4 ? 0 : off < 0 ? w << (-8 * off) : w >> (8 * off);
  }
  uint32_t w = 0;
  for (int i = 0; i < 4; i++)
    if (j + i >= 0 && j + i < n) w |= (uint32_t)gptr(row)[j + i] << (8 * i);
  return w;
}
// bit i: byte i is not 0
__device__ __forceinline__ uint32_t nonzero4(uint32_t w) {
  const uint32_t top = (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) >> 7;
  return (top & 1) | (top >> 7 & 2) | (top >> 14 & 4) | (top >> 21 & 8);
}

// A value that is infinite or NaN among the 16 bytes
template <int DT, bool Q8>
__device__ __forceinline__ bool not_finite(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (Q8) {
#pragma unroll
      for (int b = 0; b < 32; b += 8) bad |= (w[i] >> b & 0x7f) == 0x7f;
    } else {
      constexpr uint32_t E = DT == DT_F16 ? 0x7c00 : 0x7f80;
      bad |= (w[i] & E) == E || (w[i] >> 16 & E) == E;
    }
  }
  return bad;
}

// A row's sum of weights at maximum m, as one at maximum `to`.  In 8 bits the maximum is that of score and V's exponent
// together and the sum one of scores alone: it can count where 2^(m - to) is below fp32's range (64 tokens of scale
// 2^-60 before 64 of 2^93: without them twice the value), so it moves in two steps.
__device__ __forceinline__ float sum_at(float l, float m, float to) {
  const float half = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(0.5f * (m - to));
  return l * half * half;
}

// 4 results of a tile's column: channels d0 .. of row t0 + column / G, head column % G
template <int DT, int D>
__device__ __forceinline__ void put_result(const TreeArgs& a, int hk, int t0, int column, int d0, f32x4 O, float L) {
  const int G = a.hq / a.hkv;
  O *= L > 0.f || L != L ? 1.f / L : 0.f;  // (nothing seen: 0)
  *(YR_G uint64_t*)(a.out + ((size_t)(t0 + column / G) * a.hq + (size_t)hk * G + column % G) * D + d0) =
      (uint64_t)pack2<DT>(O[2], O[3]) << 32 | pack2<DT>(O[0], O[1]);
}

// Q8: a cache in e4m3.  NC: groups of 16 columns of a wave.  K and V go straight from memory
// into LDS; page ids and scales come ahead of them, a token a lane.  The loads are counted,
// so that each wait names what has to have landed.
//
// SHARE false: a tile's columns fit one wave, its tokens are split over the waves.  Each has a
// slot for K and one for V; its next K block is requested as soon as this one's fragments
// are in registers and its next V block after P V, so one of the two is always in flight.
//
// SHARE true: each wave has its own columns (rows of up to 64 NC / G tokens) and all work on
// the same block, so K and V are moved to LDS once for all of them.  The slots are a ring with
// one barrier a block.
template <int DT, bool Q8, int D, int NC, bool SHARE>
__global__ __launch_bounds__(TR_WAVES * kWave, 2) void tree_kernel(TreeArgs a) {
  constexpr int T = TR_WAVES * kWave;
  constexpr int RB = Q8 ? D : 2 * D;                   // bytes of a token's head
  constexpr int BT = tr_block(RB, SHARE);              // tokens of a block
  constexpr int SLOTS = SHARE && RB == 256 ? 2 : 4;    // of K and of V in LDS
  constexpr int CPR = RB / 16, RPI = kWave / CPR;      // chunks per row, rows per load instruction
  constexpr int NL = BT / RPI, NB = BT / 16;           // loads per operand, groups of 16 tokens
  constexpr int NSMALL = Q8 ? 3 : 1;                   // loads of a block's ids and scales
  constexpr int NP = NL / TR_WAVES;                    // a wave's share of a block's loads
  __shared__ __attribute__((aligned(16))) uint8_t s_k[SLOTS][BT * RB];
  __shared__ __attribute__((aligned(16))) uint8_t s_v[SLOTS][BT * RB];
  __shared__ __attribute__((aligned(16))) float s_ks[TR_WAVES][BT], s_ev[TR_WAVES][BT], s_iv[TR_WAVES][BT], s_fv[TR_WAVES][BT];
  __shared__ __attribute__((aligned(16))) float s_rk[Q8 && DT == DT_F16 ? TR_WAVES : 1][BT], s_rv[Q8 && DT == DT_F16 ? TR_WAVES : 1][BT];
  __shared__ __attribute__((aligned(16))) uint32_t s_small[TR_WAVES][NSMALL][kWave];  // by wave or slot: ids, scale bytes
  __shared__ float s_m[TR_WAVES][16 * NC], s_l[TR_WAVES][16 * NC];
  static_assert(16 * D * 4 <= BT * RB, "a wave's O of 16 columns fits a slot");
  static_assert(NC <= 2, "O lies over a V and a K slot");
  static_assert(NL % TR_WAVES == 0, "waves load equal shares");
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int G = a.hq / a.hkv, col = lane % 16, grp = lane / 16;
  const int cols = a.tt * G;

  // fragment offsets within a block: K's chunk of row col (groups of 16 rows add 16 RB), V's of
  // this lane's row (32 rows add 32 RB)
  uint32_t koff[RB / 64], voff[D / 16];
#pragma unroll
  for (int j = 0; j < RB / 64; j++) koff[j] = col * RB + 16 * ((4 * j + grp) ^ tk_swz<RB>(col));
  if constexpr (Q8) {
    const int e = col / 2, r0 = 16 * (e / 4) + 4 * grp + e % 4;
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) voff[dt] = r0 * RB + 16 * (dt ^ tv_swz<Q8, RB>(r0)) + 8 * (col % 2);
  } else {
    const int r0 = 4 * grp + col / 4, qc = (col % 4) / 2, qh = 8 * (col % 2);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) voff[dt] = r0 * RB + 16 * ((2 * dt + qc) ^ tv_swz<Q8, RB>(r0)) + qh;
  }
  const uint32_t tok_bytes = (uint32_t)a.hkv * RB;

  // ---- this workgroup's units
  long long units = 0, x = 0, x1 = 1;
  int parts = 1;
  SeqWork work0 = seq_work(a, lane);
  // Up to 4 kv heads share a workgroup, a wave (or two) each, where a wave has enough to do:
  // they read neighbouring bytes at about the same time (loads alone, 128 bytes a head: 5.2 TB/s
  // with a workgroup a head, 6.0 with 4 heads in one).
  bool split = a.parts > 0;  // else a tile a workgroup
  if (split) {
    long long tiles;
    units = all_units(a, work0, &tiles);
    split = tiles > a.parts || units > tiles * (TR_SHORT + TR_TILE_COST);
    if (!split && blockIdx.x == 0 && tid == 0) a.split[0].x = 0;
  }
  const bool shared = !SHARE && !(a.parts && (!split || units < (long long)TR_WAVE_BLOCKS * BT * TR_WAVES * a.parts));
  const int log_heads = shared ? a.log_heads : 0, heads = 1 << log_heads, groups = a.hkv >> log_heads;
  const int w0 = __builtin_amdgcn_readfirstlane(blockIdx.x / groups), hk0 = (blockIdx.x - w0 * groups) << log_heads;
  const int streams = TR_WAVES >> log_heads, stream = SHARE ? 0 : wave & (streams - 1);  // waves of a head
  const int hk = SHARE ? hk0 : hk0 + (wave << log_heads) / TR_WAVES;                      // this wave's
  const int most = a.parts << a.log_heads;
  if (split) {
    parts = (int)min((long long)a.parts << log_heads, max(units / (TR_MIN_BLOCKS * BT), 1ll));
    if (blockIdx.x == 0 && tid == 0) a.split[0].x = units ? parts : 0;
    if (w0 >= parts) return;
    x = part_start(units, parts, w0);
    x1 = part_start(units, parts, w0 + 1);
  }
  while (true) {
    const TileAt at = split ? find_unit(a, work0, x) : find_index(a, work0, w0);
    if (at.b >= a.r.batch) return;  // (no tile left: a tile a workgroup, or no new rows)
    const SeqRows s = at.s;
    const int i0 = at.tile * a.tt;
    const long long u0 = split ? x - at.from : 0, u1 = split ? min(x1 - at.from, at.units) : 1;
    x += u1 - u0;
    const bool whole = u1 - u0 == at.units;
    const int nt = min(a.tt, s.n - i0), t0 = s.row0 + i0, first = s.len - s.n, p0 = first + i0;  // rows, first row, its place
    // tokens that some row may see (and the page table has), those before `plain` all rows
    const int end = (int)min((long long)(a.mask ? s.len : min(s.len, p0 + nt)), (long long)s.npg * a.r.page);
    const int plain = a.mask ? first : p0 + 1;
    const int nblk = end > 0 ? (end + BT - 1) / BT : 0;
    // (a tile's first TR_TILE_COST units stand for its start and hold no blocks)
    const long long tokens = split ? max(at.units - TR_TILE_COST, 1ll) : 1;
    auto block_at = [&](long long u) __attribute__((always_inline)) -> int {
      return (int)first64((split ? max(u - TR_TILE_COST, 0ll) : u) * nblk / tokens);
    };
    const int blk0 = block_at(u0), blk1 = block_at(u1);

    // ---- this lane's query rows: its column of group c is row qi of the tile, head (column % G)
    const int col0 = SHARE ? wave * 16 * NC : 0;
    int qi[NC];
    uint4 qf[NC][D / 32];
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int cw = col0 + 16 * c + col;
      qi[c] = cw / G;
      const uint16_t* src = a.q + ((size_t)(t0 + qi[c]) * a.hq + (size_t)hk * G + cw % G) * D;
#pragma unroll
      for (int st = 0; st < D / 32; st++) {
        qf[c][st] = make_uint4(0, 0, 0, 0);
        if (qi[c] < nt) qf[c][st] = ldg16(src + (Q8 ? 16 * (4 * (st / 2) + grp) + 8 * (st % 2) : 32 * st + 8 * grp));
      }
    }

    // A block's tokens, one a lane (lane % BT): entry of the page table, then the place in the cache
    // (0 where there is none) and which lanes have one.
    struct Block {
      uint32_t place;
      uint64_t have;
    };
    auto token = [&](int blk) __attribute__((always_inline)) -> uint32_t { return (uint32_t)(min(blk, nblk) * BT + lane % BT); };
    auto entry = [&](uint32_t x) __attribute__((always_inline)) -> uint32_t {
      return (uint32_t)((uint64_t)x * a.page_mul >> a.page_shift);
    };
    auto id_at = [&](int blk) __attribute__((always_inline)) -> const int32_t* {
      return a.r.kv_indices + s.pg0 + min((int)entry(token(blk)), s.npg - 1);
    };
    auto place = [&](int blk, int id) __attribute__((always_inline)) -> Block {
      const uint32_t x = token(blk), e = entry(x);
      const bool ok = (int)x < end && (int)e < s.npg && (unsigned)id < (unsigned)a.r.num_pages;
      Block t;
      t.place = ok ? (uint32_t)id * (uint32_t)a.r.page + (x - e * (uint32_t)a.r.page) : 0;
      t.have = __ballot(ok);
      return t;
    };
    // loads u0 .. u0 + N - 1 of a block's K or V
    auto issue = [&](uint32_t where, const uint8_t* cache, uint8_t* dst, auto is_k_c, auto n_c, int u0) __attribute__((always_inline)) {
      constexpr bool IS_K = decltype(is_k_c)::value;
      const uint8_t* const base = cache + (size_t)hk * RB;
#pragma unroll
      for (int u = 0; u < decltype(n_c)::value; u++) {
        const int row = RPI * (u0 + u) + lane / CPR;
        const uint32_t from = (uint32_t)__shfl((int)where, row);
        const int chunk = (lane % CPR) ^ (IS_K ? tk_swz<RB>(row) : tv_swz<Q8, RB>(row));
        lds_load16(reinterpret_cast<const uint16_t*>(base + (uint64_t)from * tok_bytes + 16 * chunk),
                   reinterpret_cast<uint16_t*>(dst + 1024 * (u0 + u)));
      }
    };

    float m_i[NC], l_i[NC];
    bool far = false;  // some row's m_i is beyond kFarScore
    f32x4 acc[NC][D / 16];
#pragma unroll
    for (int c = 0; c < NC; c++) {
      m_i[c] = -INFINITY;
      l_i[c] = 0.f;
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) acc[c][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // Scales.  K's go into the conversion (f16 holds every code times 2^-15 to 2^7: of a scale beyond these the
    // rest multiplies the token's scores, and V's exponent follows).  V's, 2^e, are added to the scores, as e in the
    // exponent (the start of the sums that are the scores: no instruction a weight):
    //   P = 2^(x + e - m),  O += P code,  L += P 2^-e,  m the running maximum of x + e
    // so that P keeps to its type's range whatever the scales are, by each row's own maximum: a token that
    // a row does not see, or that counts little, takes no bits from it (f16 holds all of a weight's down to 2^-21 of
    // the row's largest 2^(x + e), bf16 to 2^-126).  Where a token's scale is below 2^-60 of the
    // largest so far, P may be 0 and its part in L is not: there L += 2^(x - m), in two factors like all that L is
    // multiplied by.  A scale below 2^-60 counts as that (L stays in range) and its weight takes the rest on its
    // way to O.
    int top = 0;       // the largest scale byte so far
    bool low = false;  // some token of the block has a scale for that
    bool wide = false; // some key's scale is beyond what f16 holds
    auto put_scales = [&](int kb, int vb, uint64_t have) __attribute__((always_inline)) {
      const bool ok = have >> lane & 1;
      const int e = min(max(vb, 67), 254);
      const float ev = vb == 255 ? NAN : (float)(e - 127) * a.scale_inv;
      s_ks[wave][lane % BT] = __uint_as_float((uint32_t)kb << 23);  // (what the conversion takes: 0 is 2^-127, 255 NaN)
      s_ev[wave][lane % BT] = ev;
      s_iv[wave][lane % BT] = __uint_as_float(e < 254 ? (uint32_t)(254 - e) << 23 : 0x400000u);
      s_fv[wave][lane % BT] = __uint_as_float((uint32_t)(vb - e + 127) << 23);
      low = wide = false;
      // (rare, and the first block)
      if (__builtin_amdgcn_ballot_w64(ok && (vb > top || vb < max(top - 60, 67) || (DT == DT_F16 && (unsigned)(kb - 112) > 22)))) {
        int most = ok && vb != 255 ? max(vb, top) : top;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, kWave));
        top = __builtin_amdgcn_readfirstlane(most);
        low = __builtin_amdgcn_ballot_w64(ok && vb < max(top - 60, 67)) != 0;
        if constexpr (DT == DT_F16) {
          const int held = kb == 255 ? kb : min(max(kb, 112), 134);
          wide = __builtin_amdgcn_ballot_w64(ok && kb != held) != 0;
          if (wide) {
            s_ks[wave][lane % BT] = __uint_as_float((uint32_t)held << 23);
            s_ev[wave][lane % BT] = kb != held ? 0.f : ev;
            s_rk[wave][lane % BT] = __uint_as_float((uint32_t)(kb - held + 127) << 23);
            s_rv[wave][lane % BT] = kb != held ? ev : 0.f;
          }
        }
      }
    };

    // Some row may not see some token of the block (uniform, also over waves)
    auto is_masked = [&](int blk, uint64_t have) __attribute__((always_inline)) -> bool { return (blk + 1) * BT > plain || have != ~0ull; };
    // One block for this wave's columns.  after_k: K's fragments are in registers; before_v: V
    // is needed.
    auto compute = [&](int blk, uint64_t have, const uint8_t* kt, uint8_t* vt, auto after_k, auto before_v) __attribute__((always_inline)) {
      f32x4 sc[NC][NB];
      float kscale[NB];
#pragma unroll
      for (int n = 0; n < NB; n++) {
        f32x4 start = {0.f, 0.f, 0.f, 0.f};
        if constexpr (Q8) {
          start = *reinterpret_cast<const f32x4*>(&s_ev[wave][16 * n + 4 * grp]);
          kscale[n] = s_ks[wave][16 * n + col];
        }
#pragma unroll
        for (int c = 0; c < NC; c++) sc[c][n] = start;
      }
      uint4 kw[TR_FRAGMENTS + 1];
      auto k_read = [&](int s) __attribute__((always_inline)) {
        kw[s % (TR_FRAGMENTS + 1)] = *reinterpret_cast<const uint4*>(&kt[koff[s / NB] + 16 * (s % NB) * RB]);
      };
#pragma unroll
      for (int s = 0; s < TR_FRAGMENTS; s++) k_read(s);
#pragma unroll
      for (int s = 0; s < NB * (RB / 64); s++) {
        if (s + TR_FRAGMENTS < NB * (RB / 64)) k_read(s + TR_FRAGMENTS);
        __builtin_amdgcn_sched_barrier(0);
        const int n = s % NB, j = s / NB;
        const uint4 w = kw[s % (TR_FRAGMENTS + 1)];
        if constexpr (Q8) {
          const uint2 f0 = e4m3x4<DT>(w.x, kscale[n]), f1 = e4m3x4<DT>(w.y, kscale[n]), f2 = e4m3x4<DT>(w.z, kscale[n]),
                      f3 = e4m3x4<DT>(w.w, kscale[n]);
#pragma unroll
          for (int c = 0; c < NC; c++) {
            sc[c][n] = mfma16<DT>(make_uint4(f0.x, f0.y, f1.x, f1.y), qf[c][2 * j], sc[c][n]);
            sc[c][n] = mfma16<DT>(make_uint4(f2.x, f2.y, f3.x, f3.y), qf[c][2 * j + 1], sc[c][n]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < NC; c++) sc[c][n] = mfma16<DT>(w, qf[c][j], sc[c][n]);
        }
      }
      // (the other wave of the SIMD is given way to in the softmax: its matrix instructions and these
      // vector ones then overlap; a chunk of 2048 rows after 14 K tokens 672 -> 635 us)
      __builtin_amdgcn_s_setprio(0);
      after_k();
      // mask: this lane's tokens are 16 n + 4 grp + i
      const int pos0 = blk * BT;
      const bool masked = is_masked(blk, have);
      uint32_t seen[NC];
#pragma unroll
      for (int c = 0; c < NC; c++) seen[c] = ~0u;
      if constexpr (Q8 && DT == DT_F16) {
        if (wide) {  // (uniform)
#pragma unroll
          for (int n = 0; n < NB; n++) {
            const f32x4 rest = *reinterpret_cast<const f32x4*>(&s_rk[wave][16 * n + 4 * grp]);
            const f32x4 ev = *reinterpret_cast<const f32x4*>(&s_rv[wave][16 * n + 4 * grp]);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
              for (int i = 0; i < 4; i++) sc[c][n][i] = fmaf(sc[c][n][i], rest[i], ev[i]);
          }
        }
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
          const int rel = pos0 - first, lim = (a.mask ? first : p0 + qi[c] + 1) - pos0;
          const uint8_t* const row = a.mask + (size_t)(t0 + min(qi[c], nt - 1)) * a.mask_row;
          seen[c] = 0;
          uint32_t bytes[NB];
          if (a.mask) {
#pragma unroll
            for (int n = 0; n < NB; n++) bytes[n] = mask4(row, a.mask_cols, rel + 16 * n + 4 * grp);
          }
#pragma unroll
          for (int n = 0; n < NB; n++) {
            const int x = 16 * n + 4 * grp;
            uint32_t four = (1u << min(max(lim - x, 0), 4)) - 1;
            if (a.mask) four |= nonzero4(bytes[n]);
            seen[c] |= (four & (uint32_t)(have >> x) & 15) << (4 * n);
          }
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) sc[c][n][i] = seen[c] >> (4 * n + i) & 1 ? sc[c][n][i] : -INFINITY;
        }
      }
      bool grow = false;
      float mnew[NC];
#pragma unroll
      for (int c = 0; c < NC; c++) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) mx = fmaxf(mx, sc[c][n][i]);
        mx = max_xor32(max_xor16(mx)) * a.scale_log2;
        mnew[c] = mx > m_i[c] + kLazy ? mx : m_i[c];
        grow |= mx > m_i[c] + kLazy;
      }
      if (__builtin_amdgcn_ballot_w64(grow)) {
        far = false;
#pragma unroll
        for (int c = 0; c < NC; c++) {
          const float alpha = m_i[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i[c] - mnew[c]);
          if constexpr (Q8) l_i[c] = sum_at(l_i[c], m_i[c], mnew[c]);
          else l_i[c] *= alpha;
          m_i[c] = mnew[c];
          far |= __builtin_amdgcn_ballot_w64(fabsf(m_i[c]) > kFarScore && m_i[c] > -INFINITY) != 0;
#pragma unroll
          for (int dt = 0; dt < D / 16; dt++) acc[c][dt] *= alpha;
        }
      }
      uint2 pb[NC][NB];
      auto weights = [&](auto plain_c) __attribute__((always_inline)) {
        constexpr bool PLAIN = decltype(plain_c)::value;
#pragma unroll
        for (int n = 0; n < NB; n++) {
          f32x4 iv, fv, hv;  // 2^-e; the rest of V's scale; -e / 2
          if constexpr (Q8) iv = *reinterpret_cast<const f32x4*>(&s_iv[wave][16 * n + 4 * grp]);
          if constexpr (Q8 && !PLAIN) {
            fv = *reinterpret_cast<const f32x4*>(&s_fv[wave][16 * n + 4 * grp]);
#pragma unroll
            for (int i = 0; i < 4; i++) hv[i] = 0.5f * (float)((int)(__float_as_uint(iv[i]) >> 23) - 127);
          }
#pragma unroll
          for (int c = 0; c < NC; c++) {
            const float m = m_i[c] == -INFINITY ? 0.f : m_i[c];
            f32x4 p;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              // (a row goes by its own maximum, so its weights agree)
              float x = PLAIN ? fmaf(sc[c][n][i], a.scale_log2, kPBias<DT> - m) : far_exponent(sc[c][n][i], a.scale_log2, m) + kPBias<DT>;
              p[i] = __builtin_amdgcn_exp2f(x);
              if constexpr (Q8 && !PLAIN) {
                const float root = __builtin_amdgcn_exp2f(fmaf(0.5f, x, hv[i]));
                l_i[c] = fmaf(root, root, l_i[c]);
                p[i] *= fv[i];
              } else if constexpr (Q8) {
                l_i[c] = fmaf(p[i], iv[i], l_i[c]);
              } else {
                l_i[c] += p[i];
              }
            }
            pb[c][n] = make_uint2(pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]));
          }
        }
      };
      if (far || low) weights(std::false_type{});  // (uniform)
      else weights(std::true_type{});
      __builtin_amdgcn_s_setprio(1);
      before_v();
      // Infinity or NaN in a token's V would reach the rows that do not see it as 0 * inf: such
      // tokens are left out of the product and added to those that do, one by one.
      if (masked) {
        uint64_t bad = 0;
#pragma unroll 1
        for (int u = 0; u < NL; u++) {
          const uint4 w = *reinterpret_cast<const uint4*>(vt + 1024 * u + 16 * lane);
          const uint64_t lanes = __ballot(not_finite<DT, Q8>(w));
          for (int x = 0; x < RPI; x++)
            if (lanes >> (x * CPR) & ((1ull << CPR) - 1)) bad |= 1ull << (RPI * u + x);
        }
#pragma unroll 1
        for (uint64_t left = bad; left; left &= left - 1) {
          const int x = __builtin_ctzll(left);
          const uint8_t* const row = vt + x * RB;
          const int swz = tv_swz<Q8, RB>(x);
#pragma unroll
          for (int c = 0; c < NC; c++) {
            uint2 w = make_uint2(0, 0);
#pragma unroll
            for (int n = 0; n < NB; n++)
              if (x / 16 == n) w = pb[c][n];
            const uint32_t h = x & 2 ? w.y : w.x;
            // (the lane group that holds the token tells the others; -1: not seen)
            const float mine = seen[c] >> (4 * (x / 16) + x % 4) & 1 ? (x & 1 ? hi16<DT>(h) : lo16<DT>(h)) : -1.f;
            const float p = __shfl(mine, x % 16 / 4 * 16 + col);
#pragma unroll
            for (int dt = 0; dt < D / 16; dt++) {  // channels 16 dt + 4 grp + i
              uint2 v;
              if constexpr (Q8) v = e4m3x4<DT>(*reinterpret_cast<const uint32_t*>(row + 16 * (dt ^ swz) + 4 * grp), 1.f);
              else v = *reinterpret_cast<const uint2*>(row + 16 * ((2 * dt + grp / 2) ^ swz) + 8 * (grp % 2));
              const float f[4] = {lo16<DT>(v.x), hi16<DT>(v.x), lo16<DT>(v.y), hi16<DT>(v.y)};
#pragma unroll
              for (int i = 0; i < 4; i++) acc[c][dt][i] = p < 0.f ? acc[c][dt][i] : fmaf(p, f[i], acc[c][dt][i]);
              __builtin_amdgcn_sched_barrier(0);  // (rare: no registers for it)
            }
          }
        }
        if (bad) {  // (the same for all waves of a shared block)
          if constexpr (SHARE) __syncthreads();
          if (!SHARE || wave == 0) {
            for (uint64_t left = bad; left; left &= left - 1)
              if (lane < CPR) *reinterpret_cast<uint4*>(vt + __builtin_ctzll(left) * RB + 16 * lane) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if constexpr (SHARE) __syncthreads();
        }
      }
      constexpr int DV = D / 16;
      uint4 vw[TR_FRAGMENTS + 1];
      auto v_read = [&](int s) __attribute__((always_inline)) {
        const int m = s / DV, dt = s % DV;
        uint4& to = vw[s % (TR_FRAGMENTS + 1)];
        if constexpr (Q8) {
          const uint2 w = lds_tr8(&vt[voff[dt] + 32 * m * RB]);
          to.x = w.x;
          to.y = w.y;
        } else {
          const uint2 lo = lds_tr4(reinterpret_cast<const uint16_t*>(&vt[voff[dt] + 32 * m * RB]));
          const uint2 hi = lds_tr4(reinterpret_cast<const uint16_t*>(&vt[voff[dt] + (32 * m + 16) * RB]));
          to = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      };
#pragma unroll
      for (int s = 0; s < TR_FRAGMENTS; s++) v_read(s);
#pragma unroll
      for (int s = 0; s < NB / 2 * DV; s++) {
        if (s + TR_FRAGMENTS < NB / 2 * DV) v_read(s + TR_FRAGMENTS);
        __builtin_amdgcn_sched_barrier(0);
        const int m = s / DV, dt = s % DV;
        uint4 vf = vw[s % (TR_FRAGMENTS + 1)];
        if constexpr (Q8) {
          const uint2 f0 = e4m3x4<DT>(vf.x, 1.f), f1 = e4m3x4<DT>(vf.y, 1.f);
          vf = make_uint4(f0.x, f0.y, f1.x, f1.y);
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
          acc[c][dt] = mfma16<DT>(vf, make_uint4(pb[c][2 * m].x, pb[c][2 * m].y, pb[c][2 * m + 1].x, pb[c][2 * m + 1].y),
                                  acc[c][dt]);
      }
    };

    if constexpr (!SHARE) {
      uint8_t* const ks = s_k[wave];
      uint8_t* const vs = s_v[wave];
      constexpr auto kk = std::true_type{};
      constexpr auto vv = std::false_type{};
      constexpr auto all = std::integral_constant<int, NL>{};
      Block cur, nxt;  // this block and the next
      uint32_t (*const small)[kWave] = s_small[wave];
      // The next block's scales and the ids of the one after: into LDS, like the rest, since a
      // register's load among loads into LDS is waited for with all of them.
      auto small_loads = [&](int ahead) __attribute__((always_inline)) {
        lds_load4(id_at(ahead), small[0]);
        if constexpr (Q8) {
          const size_t where = (size_t)nxt.place * a.hkv + hk;
          lds_load1(a.ks + where, small[1]);
          lds_load1(a.vs + where, small[2]);
        }
        asm volatile("" ::: "memory");
      };
      // LAST: there is no next block (a copy of its own: every path knows how many loads are in flight)
      auto consume = [&](int blk, auto last_c) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last_c)::value;
        // K has landed; V and the small loads may be on their way
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LAST ? NL : NL + NSMALL) : "memory");
        compute(
            blk, cur.have, ks, vs,
            [&]() __attribute__((always_inline)) {
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
              if constexpr (!LAST) issue(nxt.place, a.kc, ks, kk, all, 0);
            },
            [&]() __attribute__((always_inline)) {  // the small loads and the next K may be on their way
              if constexpr (!LAST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL + NSMALL) : "memory");
              else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every V fragment is in registers
        if constexpr (!LAST) {
          issue(nxt.place, a.vc, vs, vv, all, 0);
          cur = nxt;
          // the small loads of the last turn have landed
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
          const int id = (int)small[0][lane];
          if constexpr (Q8) put_scales((int)small[1][lane], (int)small[2][lane], cur.have);
          nxt = place(blk + 2 * streams, id);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          small_loads(blk + 3 * streams);
        }
      };
      // a head's waves take blocks in turn (a fixed order)
      if (blk0 + stream < blk1) {
        int blk = blk0 + stream;
        const int id0 = *gptr(id_at(blk)), id1 = *gptr(id_at(blk + streams));
        cur = place(blk, id0);
        nxt = place(blk + streams, id1);
        if constexpr (Q8) {
          const size_t where = (size_t)cur.place * a.hkv + hk;
          put_scales(gptr(a.ks)[where], gptr(a.vs)[where], cur.have);
        }
        asm volatile("" ::: "memory");
        issue(cur.place, a.kc, ks, kk, all, 0);
        issue(cur.place, a.vc, vs, vv, all, 0);
        asm volatile("" ::: "memory");
        small_loads(blk + 2 * streams);
        for (; blk + streams < blk1; blk += streams) consume(blk, std::false_type{});
        consume(blk, std::true_type{});
      }
    } else {
      constexpr int AHEAD = SLOTS - 1;
      constexpr int GROUP = 2 * NP + 1;  // a wave's loads of a block
      const int n = blk1 - blk0;
      const bool idle = nt * G <= col0;  // (no columns)
      constexpr auto share = std::integral_constant<int, NP>{};
      // block t, in slot t % SLOTS: this wave's part of K and V, its scales (one wave K's, one V's), and
      // the ids of block t + AHEAD (the others, each the same)
      auto issue_block = [&](int t, uint32_t where) __attribute__((always_inline)) {
        const int slot = t % SLOTS;
        issue(where, a.kc, s_k[slot], std::true_type{}, share, wave * NP);
        issue(where, a.vc, s_v[slot], std::false_type{}, share, wave * NP);
        const size_t head = (size_t)where * a.hkv + hk;
        if (Q8 && wave < 2) lds_load1((wave == 0 ? a.ks : a.vs) + head, s_small[slot][NSMALL > 1 ? 1 + wave : 0]);
        else lds_load4(id_at(blk0 + t + AHEAD), s_small[(t + AHEAD) % SLOTS][0]);
        asm volatile("" ::: "memory");
      };
      uint64_t have[AHEAD] = {};  // of this block and those on their way
      if (n > 0) {
        int id[AHEAD];
#pragma unroll
        for (int t = 0; t < AHEAD; t++) id[t] = *gptr(id_at(blk0 + t));
#pragma unroll
        for (int t = 0; t < AHEAD; t++) {
          const Block p = place(blk0 + t, id[t]);
          have[t] = p.have;
          if (t < n) issue_block(t, p.place);
        }
      }
      for (int t = 0; t < n; t++) {
        // this wave's part of the block has landed; those behind it may be on their way
        if (AHEAD > 2 && t + 2 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * GROUP) : "memory");
        else if (AHEAD > 1 && t + 1 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(GROUP) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // every wave's part has, and the block before is read out
        asm volatile("" ::: "memory");
        const int slot = t % SLOTS;
        int kb = 0, vb = 0;
        if constexpr (Q8) {
          kb = (int)s_small[slot][1][lane];
          vb = (int)s_small[slot][2][lane];
        }
        uint64_t have_new = 0;
        if (t + AHEAD < n) {
          const Block p = place(blk0 + t + AHEAD, (int)s_small[(t + AHEAD) % SLOTS][0][lane]);
          have_new = p.have;
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          issue_block(t + AHEAD, p.place);
        }
        if (!idle || is_masked(blk0 + t, have[0])) {  // (a masked block may need barriers)
          if constexpr (Q8) put_scales(kb, vb, have[0]);
          compute(blk0 + t, have[0], s_k[slot], s_v[slot], [] {}, [] {});
        }
#pragma unroll
        for (int u = 0; u + 1 < AHEAD; u++) have[u] = have[u + 1];
        have[AHEAD - 1] = have_new;
      }
    }

    // ---- results, or this workgroup's part of them
#pragma unroll
    for (int c = 0; c < NC; c++) {
      l_i[c] = add_xor32(add_xor16(l_i[c]));
    }
    const int rows = nt * G;
    // a part has two records: of a tile that began before it, and of one that goes on behind it
    auto record = [&](int head) __attribute__((always_inline)) -> float* {
      return a.partial + (((size_t)head * most + w0) * 2 + (u0 == 0)) * cols * (D + 4);
    };
    if (split && x >= x1 && tid == 0) {  // its last tile: the parts that this one begins, if it does
      const int n = !whole && u0 == 0 ? part_of(units, parts, x - u1 + at.units - 1) - w0 + 1 : 0;
      for (int h = hk0; h < hk0 + heads; h++) a.split[1 + (size_t)h * most + w0] = make_int4(t0, rows, n, 0);
    }
    auto put_record = [&](float* rec, int row, int d0, f32x4 v) __attribute__((always_inline)) {
      *reinterpret_cast<f32x4*>(rec + (size_t)row * (D + 4) + d0) = v;
    };
    if constexpr (SHARE) {
      float* const mine = record(hk);
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const int row = col0 + 16 * c + col;
        if (row < rows) {
          if (!whole && grp == 0) put_record(mine, row, D, f32x4{m_i[c], l_i[c], 0.f, 0.f});
#pragma unroll
          for (int dt = 0; dt < D / 16; dt++) {
            const f32x4 O = acc[c][dt];
            if (whole) put_result<DT, D>(a, hk, t0, row, 16 * dt + 4 * grp, O, l_i[c]);
            else put_record(mine, row, 16 * dt + 4 * grp, O);
          }
        }
      }
    } else {
      // the waves merge: O over each wave's own V slot (and K slot)
#pragma unroll
      for (int c = 0; c < NC; c++) {
        float* const os = reinterpret_cast<float*>(c == 0 ? s_v[wave] : s_k[wave]);
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) *reinterpret_cast<f32x4*>(os + col * D + 16 * dt + 4 * grp) = acc[c][dt];
        if (grp == 0) {
          s_m[wave][16 * c + col] = m_i[c];
          s_l[wave][16 * c + col] = l_i[c];
        }
      }
      __syncthreads();
      const int live = min(streams, blk1 - blk0);  // waves of a head that had a block
      const int quads = rows * (D / 4);
      for (int idx = tid; idx < quads * heads; idx += T) {
        const int head = idx / quads, row = idx % quads / (D / 4), d0 = idx % (D / 4) * 4, wa = head * streams;
        float M = -INFINITY, L = 0.f;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
        for (int w = wa; w < wa + live; w++) M = fmaxf(M, s_m[w][row]);
        for (int w = wa; w < wa + live; w++) {
          const float f = s_m[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][row] - M);
          const uint8_t* const os = row < 16 ? s_v[w] : s_k[w];
          const f32x4 v = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(os) + row % 16 * D + d0);
          if constexpr (Q8) L += sum_at(s_l[w][row], s_m[w][row], M);
          else L += s_l[w][row] * f;
          O += v * f;
        }
        if (whole) {
          put_result<DT, D>(a, hk0 + head, t0, row, d0, O, L);
        } else {
          put_record(record(hk0 + head), row, d0, O);
          if (d0 == 0) put_record(record(hk0 + head), row, D, f32x4{M, L, 0.f, 0.f});
        }
      }
    }

    if (x >= x1) return;
    __syncthreads();  // the slots are free again
    work0 = seq_work(a, lane);
  }
}

// Split tiles: the parts of one, 256 of its results' quads a workgroup.  Where there are fewer
// quads, SG threads share one (every SG-th part each) and meet in LDS.  (Joined by the last
// workgroup of a tile to arrive in the kernel above: 38 us for 32 rows and 32 parts; here 4 to 17.)
// TC_AHEAD of a thread's parts are on their way, where it has few TC_FEW (a chunk's, two each: 23 us for 17).
constexpr int TC_THREADS = 256, TC_AHEAD = 16, TC_FEW = 4;
template <int DT, int D>
__global__ __launch_bounds__(TC_THREADS) void tree_join_kernel(TreeArgs a) {
  const int hk = blockIdx.x % a.hkv, w0 = blockIdx.x / a.hkv, tid = threadIdx.x, most = a.parts << a.log_heads;
  const int4 at = a.split[1 + (size_t)hk * most + w0];  // first row, columns, parts
  const int items = at.y * (D / 4), item0 = blockIdx.y * TC_THREADS;
  if (w0 >= a.split[0].x || at.z == 0 || item0 >= items) return;
  const int SG = items * 2 <= TC_THREADS ? TC_THREADS / items : 1;
  const int item = SG > 1 ? tid % items : item0 + tid, j = SG > 1 ? tid / items : 0;
  const int row = item / (D / 4), d0 = item % (D / 4) * 4;
  const size_t rec = (size_t)a.tt * (a.hq / a.hkv) * (D + 4);
  const float* const base = a.partial + ((size_t)hk * most + w0) * 2 * rec + (size_t)row * (D + 4);
  float M = -INFINITY, L = 0.f;
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  const bool work = item < items && j < SG;
  auto merge = [&](auto ahead_c) __attribute__((always_inline)) {
    constexpr int AHEAD = decltype(ahead_c)::value;  // parts of this thread on their way
    for (int p = j; p < at.z; p += SG * AHEAD) {
      float2 ml[AHEAD];
      f32x4 ov[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; u++) {
        const int q = p + u * SG;
        ml[u] = make_float2(-INFINITY, 0.f);
        ov[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (q < at.z) {
          const float* const r = base + (q == 0 ? rec : 2 * rec * q);  // (the first part's is its second record)
          ml[u] = *reinterpret_cast<const float2*>(r + D);
          ov[u] = *reinterpret_cast<const f32x4*>(r + d0);
        }
      }
      float mb = M;
#pragma unroll
      for (int u = 0; u < AHEAD; u++) mb = fmaxf(mb, ml[u].x);
      const float f0 = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mb);
      L = sum_at(L, M, mb);
      O *= f0;
#pragma unroll
      for (int u = 0; u < AHEAD; u++) {
        const float f = ml[u].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[u].x - mb);
        L += sum_at(ml[u].y, ml[u].x, mb);
        O += ov[u] * f;
      }
      M = mb;
    }
  };
  if (work) {
    if (at.z <= SG * TC_FEW) merge(std::integral_constant<int, TC_FEW>{});
    else merge(std::integral_constant<int, TC_AHEAD>{});
  }
  if (SG > 1) {  // (a fixed order)
    __shared__ f32x4 so[TC_THREADS];
    __shared__ float2 sml[TC_THREADS];
    so[tid] = O;
    sml[tid] = make_float2(M, L);
    __syncthreads();
    if (j > 0) return;
    float mb = -INFINITY;
    for (int u = 0; u < SG; u++) mb = fmaxf(mb, sml[u * items + item].x);
    L = 0.f;
    O = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int u = 0; u < SG; u++) {
      const float2 v = sml[u * items + item];
      const float f = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - mb);
      L += sum_at(v.y, v.x, mb);
      O += so[u * items + item] * f;
    }
  }
  if (work) put_result<DT, D>(a, hk, at.x, row, d0, O, L);
}

// Columns of a tile, rows per tile, parts of a kv head's units (0: a tile a workgroup) of a call.
struct TreePlan {
  long long tiles;
  int nc;
  bool share;
  int tt, parts, log_heads;
};
static TreePlan tree_plan(bool ragged, int rows, int batch, int hkv, int G, int d, int max_kv_len, bool e4m3) {
  TreePlan p;
  const long long cols = ((long long)rows + batch - 1) / batch * G;  // of a sequence, on average
  p.share = cols > 32;
  p.nc = cols <= 16 || (cols > 32 && cols <= 64) ? 1 : 2;
  p.tt = ragged ? 16 * p.nc * (p.share ? TR_WAVES : 1) / G : 1;
  p.tiles = ragged ? (long long)rows / p.tt + batch : rows;
  if (p.tiles > rows) p.tiles = rows;
  const int bt = tr_block(e4m3 ? d : 2 * d, p.share);
  p.log_heads = p.share ? 0 : hkv % 4 == 0 ? 2 : hkv % 2 == 0 ? 1 : 0;
  const int target = p.share ? TR_SHARED_WG : TR_PRIVATE_WG;
  long long most = target / hkv;
  if (most < 1) most = 1;
  p.parts = (int)most;
  if (p.tiles * hkv >= TR_MANY || (max_kv_len > 0 && max_kv_len <= TR_SHORT)) {
    p.parts = 0;
    if (p.tiles * (hkv >> p.log_heads) < TR_SHARED_WG) p.log_heads = 0;
  } else if (max_kv_len > 0) {
    const long long blocks = p.tiles * (((long long)max_kv_len + TR_TILE_COST + bt - 1) / bt), need = blocks / TR_MIN_BLOCKS + 1;
    if (need < most) p.parts = (int)(need < p.tiles ? p.tiles : need);
  }
  return p;
}

}  // namespace yr

using namespace yr;

static bool tree_shape(int rows, int batch, int hq, int hkv, int d) {
  return rows > 0 && batch > 0 && hkv > 0 && hq >= hkv && hq % hkv == 0 && hq / hkv <= 16 && (d == 64 || d == 128);
}

extern "C" size_t yr_hip_gqa_tree_workspace(int rows, int batch, int ragged, int hq, int hkv, int d, int max_kv_len, int cache_dtype) {
  if (!tree_shape(rows, batch, hq, hkv, d)) return 0;
  const TreePlan p = tree_plan(ragged != 0, rows, batch, hkv, hq / hkv, d, max_kv_len, cache_dtype == YR_DTYPE_E4M3);
  if (p.parts == 0) return 0;
  return kTicketBytes + sizeof(int4) + ((size_t)p.parts << p.log_heads) * hkv * (2 * p.tt * (hq / hkv) * (d + 4) * sizeof(float) + sizeof(int4));
}

extern "C" int yr_hip_gqa_tree_plan(int rows, int batch, int ragged, int hq, int hkv, int d, int max_kv_len, int cache_dtype, int* plan3) {
  const char* nm = "yr_hip_gqa_tree_plan";
  if (!plan3 || !tree_shape(rows, batch, hq, hkv, d)) return fail(YR_E_INVALID, "%s: shape", nm);
  const TreePlan p = tree_plan(ragged != 0, rows, batch, hkv, hq / hkv, d, max_kv_len, cache_dtype == YR_DTYPE_E4M3);
  plan3[0] = 16 * p.nc * (p.share ? TR_WAVES : 1);
  plan3[1] = p.tt;
  plan3[2] = p.parts;
  return YR_OK;
}

extern "C" int yr_hip_gqa_tree_paged(const void* q, const void* k_cache, const void* v_cache, const void* k_scale,
                                     const void* v_scale, const void* tree_mask, int64_t mask_row, int mask_cols,
                                     const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                                     int n_indices, const int32_t* kv_len, void* out, int rows, int batch, int hq, int hkv,
                                     int d, int page_size, int num_pages, int max_kv_len, int cache_dtype, int dtype,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* nm = "yr_hip_gqa_tree_paged";
  TreeArgs a;
  a.r = Ragged{qo_indptr, kv_indptr, kv_indices, kv_len, rows, batch, page_size, n_indices, num_pages};
  if (!q || !k_cache || !v_cache || !out) return fail(YR_E_INVALID, "%s: null pointer", nm);
  int rc = ragged_check(nm, a.r, hq, hkv, d, dtype);
  if (rc != YR_OK) return rc;
  const bool e4m3 = cache_dtype == YR_DTYPE_E4M3;
  if (!e4m3 && cache_dtype != dtype) return fail(YR_E_INVALID, "%s: a cache is of q's type or e4m3", nm);
  if (e4m3 != (k_scale != nullptr) || e4m3 != (v_scale != nullptr))
    return fail(YR_E_INVALID, "%s: a cache in e4m3 comes with its scales, one in 16 bits without", nm);
  const int G = hq / hkv;
  if (G < 1 || G > 16) return fail(YR_E_INVALID, "%s: group size %d (1 to 16)", nm, G);
  if (tree_mask && (mask_cols < 1 || mask_row < 0)) return fail(YR_E_INVALID, "%s: tree_mask has at least one column", nm);
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15)
    return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  if (hkv > 1 << 20) return fail(YR_E_INVALID, "%s: too many heads", nm);
  if ((long long)num_pages * page_size > 0xffffffffll) return fail(YR_E_INVALID, "%s: a cache of more than 2^32 tokens", nm);
  const TreePlan p = tree_plan(qo_indptr != nullptr, rows, batch, hkv, G, d, max_kv_len, e4m3);
  const long long grid = p.parts ? (long long)p.parts * hkv : p.tiles * (hkv >> p.log_heads);
  if (grid > 0x7fffffff || (long long)rows * hkv > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
  const size_t need = yr_hip_gqa_tree_workspace(rows, batch, qo_indptr != nullptr, hq, hkv, d, max_kv_len, cache_dtype);
  if (need > workspace_bytes || (need && !workspace))
    return fail(YR_E_WORKSPACE, "%s: workspace %zu < %zu", nm, workspace_bytes, need);
  a.q = (const uint16_t*)q;
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.ks = (const uint8_t*)k_scale;
  a.vs = (const uint8_t*)v_scale;
  a.mask = (const uint8_t*)tree_mask;
  a.mask_row = mask_row;
  a.mask_cols = mask_cols;
  a.out = (uint16_t*)out;
  // (the tickets of other operators that share a workspace stay as they are)
  a.split = need ? (int4*)((char*)workspace + kTicketBytes) : nullptr;
  a.partial = need ? (float*)(a.split + 1 + ((size_t)p.parts << p.log_heads) * hkv) : nullptr;
  a.hq = hq;
  a.hkv = hkv;
  a.tt = p.tt;
  a.parts = p.parts;
  a.log_heads = p.log_heads;
  // 2^(31 + s) / page rounded up, page <= 2^s: the error is below 1 / page for x < 2^31
  int sh = 0;
  while ((1ll << sh) < page_size) sh++;
  a.page_mul = (uint32_t)(((1ull << (31 + sh)) + page_size - 1) / page_size);
  a.page_shift = 31 + sh;
  a.scale_log2 = kLog2e / sqrtf((float)d);
  a.scale_inv = 1.f / a.scale_log2;
  hipStream_t st = (hipStream_t)stream;
#define YR_TR(DT_, Q_, D_, N_, S_)                                                  \
  if (dtype == DT_ && e4m3 == Q_ && d == D_ && p.nc == N_ && p.share == S_)         \
    hipLaunchKernelGGL((tree_kernel<DT_, Q_, D_, N_, S_>), dim3((unsigned)grid), dim3(TR_WAVES * kWave), 0, st, a);
#define YR_TR2(DT_, Q_, D_) \
  YR_TR(DT_, Q_, D_, 1, false) YR_TR(DT_, Q_, D_, 2, false) YR_TR(DT_, Q_, D_, 1, true) YR_TR(DT_, Q_, D_, 2, true)
  YR_TR2(DT_F16, false, 64) YR_TR2(DT_F16, false, 128) YR_TR2(DT_F16, true, 64) YR_TR2(DT_F16, true, 128)
  YR_TR2(DT_BF16, false, 64) YR_TR2(DT_BF16, false, 128) YR_TR2(DT_BF16, true, 64) YR_TR2(DT_BF16, true, 128)
#undef YR_TR2
#undef YR_TR
  YR_CHECK_LAUNCH(nm);
  if (p.parts) {
    const dim3 joins((unsigned)((p.parts << p.log_heads) * hkv), (unsigned)((p.tt * G * (d / 4) + TC_THREADS - 1) / TC_THREADS));
#define YR_TJ(DT_, D_) \
  if (dtype == DT_ && d == D_) hipLaunchKernelGGL((tree_join_kernel<DT_, D_>), joins, dim3(TC_THREADS), 0, st, a);
    YR_TJ(DT_F16, 64) YR_TJ(DT_F16, 128) YR_TJ(DT_BF16, 64) YR_TJ(DT_BF16, 128)
#undef YR_TJ
  }
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
