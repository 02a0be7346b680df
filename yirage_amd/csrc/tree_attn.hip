// GQA attention of new rows (single tokens, trees of drafted tokens, chunks of prompts)
// over a paged cache in 16 bits or in e4m3 with a power of two per token and head.
//
//   out[t] = sum_j p_j v_j / sum_j p_j,  p_j = exp(q_t k_j / sqrt(D))
//
// over the tokens before the sequence's new ones, and of the new ones those at or before
// row t's place, or those that tree_mask[t] names.
//
// A tile is up to 16 NC / G consecutive rows of one sequence with their G heads (the
// columns of the products, which are transposed: S^T = K Q^T and O^T += V^T P^T on MFMA
// 16x16x32; a lane holds one query row of each 16).  The tile's tokens are split over
// workgroups and their waves; each wave streams its blocks through LDS slots of its own,
// with an online softmax, and waves and splits merge at the end.
//
// In 8 bits a fragment is converted between LDS and MFMA.  The conversion multiplies by
// a power of two, so a key is read with its scale for nothing and, in bf16, without
// rounding; a fragment of V holds 8 tokens, whose scales go onto the weights instead.
#include <type_traits>

#include "attn_device.h"
#include "ragged.h"

namespace yr {

constexpr int TR_WAVES = 4;
constexpr int TR_TARGET_WG = 512;  // two per CU
constexpr int TR_MIN_BLOCKS = 4;   // of a split

struct TreeArgs {
  Ragged r;
  const uint16_t* q;    // [rows][hq][D]
  const uint8_t* kc;    // [pages][page][hkv][D], 16 or 8 bits
  const uint8_t* vc;
  const uint8_t* ks;    // [pages][page][hkv] (8 bits)
  const uint8_t* vs;
  const uint8_t* mask;  // [rows][mask_cols], rows mask_row apart, or null
  uint16_t* out;
  float* partial;       // [tiles][hkv][splits][tt G][D + 4]: O, m, l
  uint32_t* tickets;    // [tiles][hkv]
  long long mask_row;
  int mask_cols, hq, hkv, tt, splits;  // tt: rows per tile
  uint32_t page_mul, page_shift;       // x / page = x page_mul >> page_shift for x < 2^31
  float scale_log2;
};

// Tile `tile` of a batch cut into tiles of up to `rows` rows of one sequence: the sequence
// (batch: none) and the tile's first row within it.  64 sequences at a time, each wave for
// itself.
__device__ __forceinline__ int2 seek_tile(const Ragged& r, int tile, int rows) {
  if (!r.qo_indptr) return make_int2(tile, 0);
  const int lane = threadIdx.x % kWave;
  int left = tile;
  for (int b = 0; b < r.batch; b += kWave) {
    int n = 0;
    if (b + lane < r.batch) {
      const int row0 = min(max(gptr(r.qo_indptr)[b + lane], 0), r.rows);
      n = (min(max(gptr(r.qo_indptr)[b + lane + 1], row0), r.rows) - row0 + rows - 1) / rows;
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int v = __shfl_up(sum, o);
      if (lane >= o) sum += v;
    }
    const uint64_t past = __ballot(sum > left);
    if (past) {
      const int i = __builtin_ctzll(past);
      return make_int2(b + i, (left - __builtin_amdgcn_readlane(sum - n, i)) * rows);
    }
    left -= __builtin_amdgcn_readlane(sum, kWave - 1);
  }
  return make_int2(r.batch, 0);
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

// Q8: a cache in e4m3.  NC: groups of 16 columns of a wave.
//
// K and V go straight into the wave's LDS slots; its next K block is requested as soon as
// this one's fragments are in registers and its next V block after P V, so one of the two
// is always in flight.  Page ids and scales come two blocks ahead, in registers, a token a
// lane; the loads of a block are counted, so that each wait names what has to have landed.
template <int DT, bool Q8, int D, int NC>
__global__ __launch_bounds__(TR_WAVES * kWave, 2) void tree_kernel(TreeArgs a) {
  constexpr int T = TR_WAVES * kWave;
  constexpr int RB = Q8 ? D : 2 * D;                   // bytes of a token's head
  constexpr int BT = 8192 / RB < 64 ? 8192 / RB : 64;  // tokens of a block
  constexpr int CPR = RB / 16, RPI = kWave / CPR;      // chunks per row, rows per load instruction
  constexpr int NL = BT / RPI, NB = BT / 16;           // loads per operand, groups of 16 tokens
  constexpr int NSMALL = Q8 ? 3 : 1;                   // loads of a block's scales and ids
  constexpr int DTV = Q8 ? DT_BF16 : DT;               // type of V and P in the second product
  __shared__ __attribute__((aligned(16))) uint8_t s_k[TR_WAVES][BT * RB];
  __shared__ __attribute__((aligned(16))) uint8_t s_v[TR_WAVES][BT * RB];
  __shared__ __attribute__((aligned(16))) float s_ks[TR_WAVES][BT], s_vs[TR_WAVES][BT];
  __shared__ float s_m[TR_WAVES][16 * NC], s_l[TR_WAVES][16 * NC];
  static_assert(16 * D * 4 <= BT * RB, "a wave's O of 16 columns fits a slot");
  static_assert(NC <= 2, "O lies over a V and a K slot");
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int hk = blockIdx.x % a.hkv, rest = blockIdx.x / a.hkv;
  const int split = rest % a.splits, tile = rest / a.splits, pair = tile * a.hkv + hk;
  const int G = a.hq / a.hkv, col = lane % 16, grp = lane / 16;

  const int2 at = seek_tile(a.r, tile, a.tt);
  const int b = __builtin_amdgcn_readfirstlane(at.x), i0 = __builtin_amdgcn_readfirstlane(at.y);
  if (b >= a.r.batch) return;
  const SeqRows s = seq_rows(a.r, b);
  const int nt = min(a.tt, s.n - i0), t0 = s.row0 + i0, first = s.len - s.n, p0 = first + i0;  // rows, first row, its place
  // tokens that some row may see (and the page table has)
  const int end = (int)min((long long)(a.mask ? s.len : min(s.len, p0 + nt)), (long long)s.npg * a.r.page);
  const int plain = a.mask ? first : p0 + 1;             // tokens before this one are seen by all

  // ---- this lane's query rows: column 16 c + col = row i of the tile, head g
  int qi[NC];
  uint4 qf[NC][D / 32];
#pragma unroll
  for (int c = 0; c < NC; c++) {
    const int qg = (16 * c + col) % G;
    qi[c] = (16 * c + col) / G;
    const uint16_t* src = a.q + ((size_t)(t0 + qi[c]) * a.hq + (size_t)hk * G + qg) * D;
#pragma unroll
    for (int st = 0; st < D / 32; st++) {
      qf[c][st] = make_uint4(0, 0, 0, 0);
      if (qi[c] < nt) qf[c][st] = ldg16(src + (Q8 ? 16 * (4 * (st / 2) + grp) + 8 * (st % 2) : 32 * st + 8 * grp));
    }
  }
  const int nblk = end > 0 ? (end + BT - 1) / BT : 0;
  const int per = (nblk + a.splits - 1) / a.splits;
  const int blk0 = min(split * per, nblk), blk1 = min(blk0 + per, nblk);

  uint8_t* const ks = s_k[wave];
  uint8_t* const vs = s_v[wave];
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

  // A block's tokens, one a lane (lane % BT): entry of the page table, then the place in the cache
  // (0 where there is none) and which lanes have one.
  struct Block {
    uint32_t place;
    uint64_t have;
  };
  auto token = [&](int blk) __attribute__((always_inline)) -> uint32_t { return (uint32_t)(blk * BT + lane % BT); };
  auto entry = [&](uint32_t x) __attribute__((always_inline)) -> uint32_t {
    return (uint32_t)((uint64_t)x * a.page_mul >> a.page_shift);
  };
  auto load_id = [&](int blk) __attribute__((always_inline)) -> int {
    return gptr(a.r.kv_indices)[s.pg0 + min((int)entry(token(min(blk, nblk))), s.npg - 1)];
  };
  auto place = [&](int blk, int id) __attribute__((always_inline)) -> Block {
    const uint32_t x = token(min(blk, nblk)), e = entry(x);
    const bool ok = (int)x < end && (int)e < s.npg && (unsigned)id < (unsigned)a.r.num_pages;
    Block t;
    t.place = ok ? (uint32_t)id * (uint32_t)a.r.page + (x - e * (uint32_t)a.r.page) : 0;
    t.have = __ballot(ok);
    return t;
  };
  const size_t tok_bytes = (size_t)a.hkv * RB;
  auto issue = [&](uint32_t where, auto is_k_c) __attribute__((always_inline)) {
    constexpr bool IS_K = decltype(is_k_c)::value;
    const uint8_t* const base = (IS_K ? a.kc : a.vc) + (size_t)hk * RB;
    uint8_t* const dst = IS_K ? ks : vs;
#pragma unroll
    for (int u = 0; u < NL; u++) {
      const int row = RPI * u + lane / CPR;
      const uint32_t from = (uint32_t)__shfl((int)where, row);
      const int chunk = (lane % CPR) ^ (IS_K ? tk_swz<RB>(row) : tv_swz<Q8, RB>(row));
      lds_load16(reinterpret_cast<const uint16_t*>(base + from * tok_bytes + 16 * chunk),
                 reinterpret_cast<uint16_t*>(dst + 1024 * u));
    }
  };
  auto scale = [&](const uint8_t* p, uint32_t where) __attribute__((always_inline)) -> uint32_t {
    return gptr(p)[(size_t)where * a.hkv + hk];
  };
  auto scale_value = [](uint32_t byte) __attribute__((always_inline)) -> float {
    return byte == 255 ? NAN : __uint_as_float(byte << 23);
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

  Block cur, nxt;                                // this block and the next
  uint32_t kb = 0, vb = 0, kb_next = 0, vb_next = 0;  // their scales
  int id_ahead = 0;                              // of the block after
  // LAST: there is no next block (a copy of its own: every path knows how many loads are in flight)
  auto consume = [&](int blk, auto last_c) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(last_c)::value;
    // K has landed; V and the small loads may be on their way
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LAST ? NL : NL + NSMALL) : "memory");
    if constexpr (Q8) {
      s_ks[wave][lane % BT] = scale_value(kb);
      s_vs[wave][lane % BT] = scale_value(vb);
      asm volatile("" ::: "memory");
    }
    f32x4 sc[NC][NB];
#pragma unroll
    for (int n = 0; n < NB; n++) {
#pragma unroll
      for (int c = 0; c < NC; c++) sc[c][n] = f32x4{0.f, 0.f, 0.f, 0.f};
      float kscale = 1.f;
      if constexpr (Q8) kscale = s_ks[wave][16 * n + col];
#pragma unroll
      for (int j = 0; j < RB / 64; j++) {
        const uint4 w = *reinterpret_cast<const uint4*>(&ks[koff[j] + 16 * n * RB]);
        if constexpr (Q8) {
          const uint2 f0 = e4m3x4<DT>(w.x, kscale), f1 = e4m3x4<DT>(w.y, kscale), f2 = e4m3x4<DT>(w.z, kscale),
                      f3 = e4m3x4<DT>(w.w, kscale);
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
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every K fragment is in registers
    if constexpr (!LAST) issue(nxt.place, std::true_type{});
    // mask: this lane's tokens are 16 n + 4 grp + i
    const int pos0 = blk * BT;
    const bool masked = pos0 + BT > plain || cur.have != ~0ull;  // (uniform)
    uint32_t seen[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) seen[c] = ~0u;
    if (masked) {
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const int rel = pos0 - first, lim = (a.mask ? first : p0 + qi[c] + 1) - pos0;
        const uint8_t* const row = a.mask + (size_t)(t0 + min(qi[c], nt - 1)) * a.mask_row;
        seen[c] = 0;
#pragma unroll 1
        for (int e = 0; e < 4 * NB; e++) {
          const int x = 16 * (e / 4) + 4 * grp + e % 4;
          bool ok = x < lim;
          if (a.mask && !ok && rel + x < a.mask_cols) ok = gptr(row)[rel + x] != 0;
          if (ok && (cur.have >> x & 1)) seen[c] |= 1u << e;
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
        m_i[c] = mnew[c];
        far |= __builtin_amdgcn_ballot_w64(fabsf(m_i[c]) > kFarScore && m_i[c] > -INFINITY) != 0;
        l_i[c] *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) acc[c][dt] *= alpha;
      }
    }
    f32x4 vscale[NB];
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < NB; n++) vscale[n] = *reinterpret_cast<const f32x4*>(&s_vs[wave][16 * n + 4 * grp]);
    }
    uint2 pb[NC][NB];
#pragma unroll
    for (int c = 0; c < NC; c++) {
      float mref = m_i[c] == -INFINITY ? 0.f : m_i[c], scl = a.scale_log2;
      if (far) {  // (uniform; a row goes by its own maximum, so its weights agree)
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) sc[c][n][i] = far_exponent(sc[c][n][i], scl, mref);
        mref = 0.f;
        scl = 1.f;
      }
      mref -= kPBias<DTV>;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        f32x4 p;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(sc[c][n][i], scl, -mref));
          l_i[c] += p[i];
          if constexpr (Q8) p[i] *= vscale[n][i];
        }
        if (Q8 && masked) {  // an unseen token's scale may be NaN
#pragma unroll
          for (int i = 0; i < 4; i++) p[i] = seen[c] >> (4 * n + i) & 1 ? p[i] : 0.f;
        }
        pb[c][n] = make_uint2(pack2<DTV>(p[0], p[1]), pack2<DTV>(p[2], p[3]));
      }
    }
    // V has landed; the small loads and the next K may be on their way
    if constexpr (!LAST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL + NSMALL) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // Infinity or NaN in a token's V would reach the rows that do not see it as 0 * inf: such
    // tokens leave the block and are added to those that do, one by one.
    if (masked) {
      uint64_t bad = 0;
#pragma unroll 1
      for (int u = 0; u < NL; u++) {
        const uint4 w = *reinterpret_cast<const uint4*>(vs + 1024 * u + 16 * lane);
        const uint64_t lanes = __ballot(not_finite<DT, Q8>(w));
        for (int x = 0; x < RPI; x++)
          if (lanes >> (x * CPR) & (CPR == 64 ? ~0ull : (1ull << CPR) - 1)) bad |= 1ull << (RPI * u + x);
      }
      for (; bad; bad &= bad - 1) {
        const int x = __builtin_ctzll(bad);
        const uint8_t* const row = vs + x * RB;
        const int swz = tv_swz<Q8, RB>(x);
#pragma unroll
        for (int c = 0; c < NC; c++) {
          uint2 w = make_uint2(0, 0);
#pragma unroll
          for (int n = 0; n < NB; n++)
            if (x / 16 == n) w = pb[c][n];
          const uint32_t h = x & 2 ? w.y : w.x;
          // (the lane group that holds the token tells the others; -1: not seen)
          const float mine = seen[c] >> (4 * (x / 16) + x % 4) & 1 ? (x & 1 ? hi16<DTV>(h) : lo16<DTV>(h)) : -1.f;
          const float p = __shfl(mine, x % 16 / 4 * 16 + col);
#pragma unroll
          for (int dt = 0; dt < D / 16; dt++) {  // channels 16 dt + 4 grp + i
            uint2 v;
            if constexpr (Q8) v = e4m3x4<DT_BF16>(*reinterpret_cast<const uint32_t*>(row + 16 * (dt ^ swz) + 4 * grp), 1.f);
            else v = *reinterpret_cast<const uint2*>(row + 16 * ((2 * dt + grp / 2) ^ swz) + 8 * (grp % 2));
            const float f[4] = {lo16<DTV>(v.x), hi16<DTV>(v.x), lo16<DTV>(v.y), hi16<DTV>(v.y)};
#pragma unroll
            for (int i = 0; i < 4; i++) acc[c][dt][i] = p < 0.f ? acc[c][dt][i] : fmaf(p, f[i], acc[c][dt][i]);
            __builtin_amdgcn_sched_barrier(0);  // (rare: no registers for it)
          }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (lane < CPR) *reinterpret_cast<uint4*>(vs + x * RB + 16 * lane) = make_uint4(0, 0, 0, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
#pragma unroll
    for (int m = 0; m < NB / 2; m++)
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) {
        uint4 vf;
        if constexpr (Q8) {
          const uint2 w = lds_tr8(&vs[voff[dt] + 32 * m * RB]);
          const uint2 f0 = e4m3x4<DTV>(w.x, 1.f), f1 = e4m3x4<DTV>(w.y, 1.f);
          vf = make_uint4(f0.x, f0.y, f1.x, f1.y);
        } else {
          const uint2 lo = lds_tr4(reinterpret_cast<const uint16_t*>(&vs[voff[dt] + 32 * m * RB]));
          const uint2 hi = lds_tr4(reinterpret_cast<const uint16_t*>(&vs[voff[dt] + (32 * m + 16) * RB]));
          vf = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
          acc[c][dt] = mfma16<DTV>(vf, make_uint4(pb[c][2 * m].x, pb[c][2 * m].y, pb[c][2 * m + 1].x, pb[c][2 * m + 1].y),
                                   acc[c][dt]);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every V fragment is in registers
    if constexpr (!LAST) {
      issue(nxt.place, std::false_type{});
      cur = nxt;
      kb = kb_next;
      vb = vb_next;
      nxt = place(blk + 2 * TR_WAVES, id_ahead);
      asm volatile("" ::: "memory");
      if constexpr (Q8) {
        kb_next = scale(a.ks, nxt.place);
        vb_next = scale(a.vs, nxt.place);
      }
      id_ahead = load_id(blk + 3 * TR_WAVES);
      asm volatile("" ::: "memory");
    }
  };
  // wave w takes blocks w, w + TR_WAVES, .. of the split (a fixed order)
  if (blk0 + wave < blk1) {
    int blk = blk0 + wave;
    const int id0 = load_id(blk), id1 = load_id(blk + TR_WAVES);
    cur = place(blk, id0);
    nxt = place(blk + TR_WAVES, id1);
    if constexpr (Q8) {
      kb = scale(a.ks, cur.place);
      vb = scale(a.vs, cur.place);
    }
    asm volatile("" ::: "memory");
    issue(cur.place, std::true_type{});
    issue(cur.place, std::false_type{});
    asm volatile("" ::: "memory");
    if constexpr (Q8) {
      kb_next = scale(a.ks, nxt.place);
      vb_next = scale(a.vs, nxt.place);
    }
    id_ahead = load_id(blk + 2 * TR_WAVES);
    asm volatile("" ::: "memory");
    for (; blk + TR_WAVES < blk1; blk += TR_WAVES) consume(blk, std::false_type{});
    consume(blk, std::true_type{});
  }

  // ---- the waves merge: O over each wave's own V slot (and K slot)
#pragma unroll
  for (int c = 0; c < NC; c++) {
    l_i[c] = add_xor32(add_xor16(l_i[c]));
    float* const os = reinterpret_cast<float*>(c == 0 ? vs : ks);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) *reinterpret_cast<f32x4*>(os + col * D + 16 * dt + 4 * grp) = acc[c][dt];
    if (grp == 0) {
      s_m[wave][16 * c + col] = m_i[c];
      s_l[wave][16 * c + col] = l_i[c];
    }
  }
  __syncthreads();
  const int live = min(TR_WAVES, blk1 - blk0);  // waves that had a block
  const int rows = nt * G;
  for (int idx = tid; idx < rows * (D / 4); idx += T) {
    const int row = idx / (D / 4), d0 = idx % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < live; w++) M = fmaxf(M, s_m[w][row]);
    for (int w = 0; w < live; w++) {
      const float f = s_m[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][row] - M);
      const uint8_t* const os = row < 16 ? s_v[w] : s_k[w];
      const f32x4 v = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(os) + row % 16 * D + d0);
      L += s_l[w][row] * f;
      O += v * f;
    }
    if (a.splits == 1) {
      const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
      O *= inv;
      *(YR_G uint64_t*)(a.out + ((size_t)(t0 + row / G) * a.hq + (size_t)hk * G + row % G) * D + d0) =
          (uint64_t)pack2<DT>(O[2], O[3]) << 32 | pack2<DT>(O[0], O[1]);
    } else {
      float* rec = a.partial + (((size_t)pair * a.splits + split) * a.tt * G + row) * (D + 4);
      st_agent4(rec + d0, make_float4(O[0], O[1], O[2], O[3]));
      if (d0 == 0) st_agent4(rec + D, make_float4(M, L, 0.f, 0.f));
    }
  }
  if (a.splits == 1) return;

  // ---- the splits meet in the workgroup that arrives last: a thread takes 4 dims of one row
  // over every SG-th split, 8 records in flight, and the SG parts meet in LDS (a fixed order)
  if (!arrive_last(&a.tickets[pair], a.splits)) return;
  constexpr int MU = 8;
  const int items = rows * (D / 4);
  const int SG = items * 2 <= T ? T / items : 1;
  f32x4* const so = reinterpret_cast<f32x4*>(&s_v[0][0]);
  float2* const sml = reinterpret_cast<float2*>(&s_k[0][0]);
  for (int item0 = 0; item0 < items; item0 += T) {  // (one turn where SG > 1)
    const int item = SG > 1 ? tid % items : item0 + tid, j = SG > 1 ? tid / items : 0;
    const int row = item / (D / 4), d0 = item % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    const bool work = item < items && j < SG;
    if (work) {
      const float* base = a.partial + ((size_t)pair * a.splits * a.tt * G + row) * (D + 4);
      const size_t next = (size_t)a.tt * G * (D + 4);
      for (int s0 = j; s0 < a.splits; s0 += SG * MU) {
        float4 ml[MU], ov[MU];
#pragma unroll
        for (int u = 0; u < MU; u++) {
          ml[u] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
          ov[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (s0 + u * SG < a.splits) {
            ml[u] = ld_agent4(base + (size_t)(s0 + u * SG) * next + D);
            ov[u] = ld_agent4(base + (size_t)(s0 + u * SG) * next + d0);
          }
        }
        float mb = M;
#pragma unroll
        for (int u = 0; u < MU; u++) mb = fmaxf(mb, ml[u].x);
        const float f0 = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mb);
        L *= f0;
        O *= f0;
#pragma unroll
        for (int u = 0; u < MU; u++) {
          const float f = ml[u].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[u].x - mb);
          L += ml[u].y * f;
          O += f32x4{ov[u].x, ov[u].y, ov[u].z, ov[u].w} * f;
        }
        M = mb;
      }
    }
    if (SG > 1) {
      if (work) {
        so[j * items + item] = O;
        if (d0 == 0) sml[j * 16 * NC + row] = make_float2(M, L);
      }
      __syncthreads();
      if (!work || j > 0) return;
      float mb = -INFINITY;
      for (int u = 0; u < SG; u++) mb = fmaxf(mb, sml[u * 16 * NC + row].x);
      L = 0.f;
      O = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int u = 0; u < SG; u++) {
        const float2 v = sml[u * 16 * NC + row];
        const float f = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - mb);
        L += v.y * f;
        O += so[u * items + item] * f;
      }
    }
    if (work) {
      const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
      O *= inv;
      *(YR_G uint64_t*)(a.out + ((size_t)(t0 + row / G) * a.hq + (size_t)hk * G + row % G) * D + d0) =
          (uint64_t)pack2<DT>(O[2], O[3]) << 32 | pack2<DT>(O[0], O[1]);
    }
  }
}

// Groups of 16 columns, rows per tile, tiles and splits of a call.
struct TreePlan {
  long long tiles;
  int nc, tt, splits;
};
static TreePlan tree_plan(bool ragged, int rows, int batch, int hkv, int G, int d, int max_kv_len, bool e4m3) {
  TreePlan p;
  const long long cols = ((long long)rows + batch - 1) / batch * G;  // of a sequence, on average
  p.nc = cols <= 16 ? 1 : 2;
  p.tt = ragged ? 16 * p.nc / G : 1;
  p.tiles = ragged ? (long long)rows / p.tt + batch : rows;
  if (p.tiles > rows) p.tiles = rows;
  const int rb = e4m3 ? d : 2 * d, bt = 8192 / rb < 64 ? 8192 / rb : 64;
  const long long pairs = p.tiles * hkv, blocks = ((long long)max_kv_len + bt - 1) / bt;
  long long sp = (TR_TARGET_WG + pairs - 1) / pairs;
  if (sp > blocks / TR_MIN_BLOCKS) sp = blocks / TR_MIN_BLOCKS;
  if (pairs > kMaxTickets || sp < 1) sp = 1;
  p.splits = (int)sp;
  return p;
}

}  // namespace yr

using namespace yr;

extern "C" size_t yr_hip_gqa_tree_workspace(int rows, int batch, int ragged, int hq, int hkv, int d, int max_kv_len, int cache_dtype) {
  if (rows <= 0 || batch <= 0 || hkv <= 0 || hq < hkv || hq % hkv || hq / hkv > 16 || d <= 0 || max_kv_len <= 0) return 0;
  const TreePlan p = tree_plan(ragged != 0, rows, batch, hkv, hq / hkv, d, max_kv_len, cache_dtype == YR_DTYPE_E4M3);
  if (p.splits == 1) return 0;
  return kTicketBytes + (size_t)p.tiles * hkv * p.splits * p.tt * (hq / hkv) * (d + 4) * sizeof(float);
}

extern "C" int yr_hip_gqa_tree_plan(int rows, int batch, int ragged, int hq, int hkv, int d, int max_kv_len, int cache_dtype, int* plan3) {
  const char* nm = "yr_hip_gqa_tree_plan";
  if (!plan3 || rows <= 0 || batch <= 0 || hkv <= 0 || hq < hkv || hq % hkv || hq / hkv > 16 || d <= 0 || max_kv_len <= 0)
    return fail(YR_E_INVALID, "%s: shape", nm);
  const TreePlan p = tree_plan(ragged != 0, rows, batch, hkv, hq / hkv, d, max_kv_len, cache_dtype == YR_DTYPE_E4M3);
  plan3[0] = p.nc;
  plan3[1] = p.tt;
  plan3[2] = p.splits;
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
  if (max_kv_len <= 0) return fail(YR_E_INVALID, "%s: max_kv_len must be positive", nm);
  if (tree_mask && (mask_cols < 1 || mask_row < 0)) return fail(YR_E_INVALID, "%s: tree_mask has at least one column", nm);
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15)
    return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  if ((long long)num_pages * page_size > 0xffffffffll) return fail(YR_E_INVALID, "%s: a cache of more than 2^32 tokens", nm);
  const TreePlan p = tree_plan(qo_indptr != nullptr, rows, batch, hkv, G, d, max_kv_len, e4m3);
  if (p.tiles * hkv * p.splits > 0x7fffffff || (long long)rows * hkv > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
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
  a.tickets = (uint32_t*)workspace;
  a.partial = need ? (float*)((char*)workspace + kTicketBytes) : nullptr;
  a.hq = hq;
  a.hkv = hkv;
  a.tt = p.tt;
  a.splits = p.splits;
  // 2^(31 + s) / page rounded up, page <= 2^s: the error is below 1 / page for x < 2^31
  int sh = 0;
  while ((1ll << sh) < page_size) sh++;
  a.page_mul = (uint32_t)(((1ull << (31 + sh)) + page_size - 1) / page_size);
  a.page_shift = 31 + sh;
  a.scale_log2 = kLog2e / sqrtf((float)d);
  const unsigned grid = (unsigned)(p.tiles * hkv * p.splits);
  hipStream_t st = (hipStream_t)stream;
#define YR_TR(DT_, Q_, D_, N_)                                  \
  if (dtype == DT_ && e4m3 == Q_ && d == D_ && p.nc == N_)      \
    hipLaunchKernelGGL((tree_kernel<DT_, Q_, D_, N_>), dim3(grid), dim3(TR_WAVES * kWave), 0, st, a);
#define YR_TR2(DT_, Q_) YR_TR(DT_, Q_, 64, 1) YR_TR(DT_, Q_, 64, 2) YR_TR(DT_, Q_, 128, 1) YR_TR(DT_, Q_, 128, 2)
  YR_TR2(DT_F16, false) YR_TR2(DT_F16, true) YR_TR2(DT_BF16, false) YR_TR2(DT_BF16, true)
#undef YR_TR2
#undef YR_TR
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
