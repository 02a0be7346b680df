// GQA attention over selected pages of a paged cache: row t of kv head h
// attends to the tokens at or before its position in the pages listed for
// (t, h).
//
// A tile is up to 16 / G consecutive rows of one sequence (16 query rows of one
// kv head with their G heads, an MFMA's 16 columns).  Its workgroup forms the
// union of the rows' lists, each page with a mask of the rows that chose it, so
// a page that several rows share is read once and none costs more than in a
// tile of its own.  The waves take 32-token blocks of the union's tokens in
// turn, each with an online softmax, and merge at the end.
//
// The contractions are transposed: S^T = K Q^T and O^T += V^T P^T on MFMA
// 16x16x32.  A lane then holds one query row (its column) and 8 of the block's
// 32 tokens: the row maximum is 7 comparisons and two permlane swaps, and P^T is
// already the B operand of the second product (k slots 8 g + 4 j + i of lane
// group g carry tokens 16 j + 4 g + i), while V^T comes from row-major V by
// transposing reads in that same order.
//
// A decode step is bound by memory and its chain of dependent loads: 32 rows of 128
// pages of 16, 8 kv heads of 64 (134 MB) 25 us, 5.3 TB/s; one row of 32 pages of 64,
// d = 128, 12 us, of which the lists 3, the blocks 3, the merges of waves and splits
// 6.  Many rows are bound by what moves from L2 to LDS: 777 rows of 16 pages of 64, 8
// kv heads of 4 heads of 128, 107 us, 1.8 GB of unions, 17 TB/s.  (Repeated inputs, one
// call after another.)
#include <type_traits>

#include "attn_device.h"
#include "ragged.h"

namespace yr {

constexpr int SP_WAVES = 4;           // (8: 32 rows of 64 pages of 16, d = 128: 26.1 for 25.4 us; 64 of 16 22.1 for 16.4)
constexpr int SP_BLK = 32;            // tokens per wave block
constexpr int SP_MAX_ENTRIES = 1024;  // list entries of a tile
constexpr int SP_TARGET_WG = 256;     // one per CU (512: 4 rows of 32 pages of 64 17.6 us for 14.2, 32 of 64 of 16 30.3 for 25.1)
constexpr int SP_MIN_BLOCKS = 4;      // blocks per split at least (1 row of 32 pages of 64: 2 16.7 us, 4 13.3, 8 12.4; of 8 pages 10.8, 10.4, 11.4)

struct SparseArgs {
  Ragged r;
  const uint16_t* q;      // [rows][hq][D]
  const uint16_t* kc;     // [pages][page][hkv][D]
  const uint16_t* vc;
  const int32_t* pages;   // [rows][hkv][top]
  uint16_t* out;
  float* partial;         // [tiles][hkv][splits][tt G][D + 4]: O, m, l
  uint32_t* tickets;      // [tiles][hkv]
  int hq, hkv, top, tt, splits;  // tt: rows per tile
  float scale_log2;
};

// P is rounded to 16 bits for the second product, the row sum is not: half a step of
// each weight, against the result's own half step (fp32 products would take 8 times
// the matrix instructions).  f16's normal range ends at
// 2^-14: weights carry a factor 2^7 there (cancelled by the row sum, at most
// 2^15 with the lazy maximum's slack of 2^8), so a weight loses bits only below
// 2^-21 of the largest and vanishes below 2^-32.
template <int DT>
constexpr float kPBias = DT == DT_F16 ? 7.f : 0.f;

// An exponent is one fma, score log2 e / sqrt(D) less the running maximum, a rounded
// number: the largest comes out as that rounding, a 16th at most up to here.  From
// 2^24 on it may be 1 and more, and P, up to 2^15 with its factor and slack, would leave
// f16's range, from 2^31 on fp32's; so beyond this the product is rounded like the
// maximum before they are subtracted (777 rows of 16 pages of 64: 1 % for the branch).
constexpr float kFarScore = 0x1p20f;
__device__ __forceinline__ float far_exponent(float score, float scale, float m) {
  float x = score * scale;
  asm volatile("" : "+v"(x));  // (no fma)
  return fabsf(m) > kFarScore ? x - m : fmaf(score, scale, -m);
}

// 16-byte chunk permutations of an LDS row of D elements.  K fragments read one
// chunk column of 16 consecutive rows, transposing V reads a chunk pair of 4
// consecutive rows: any 8 lanes of either hit 8 chunks apart modulo 128 bytes.
template <int D>
__device__ __forceinline__ int k_swz(int row) { return row & (D == 128 ? 15 : 7); }
template <int D>
__device__ __forceinline__ int v_swz(int row) {
  return D == 128 ? ((row & 7) << 1) | ((row >> 3) & 1) : (row & 3) << 1;
}

// Union of the lists of rows t0 .. t0 + nt - 1 (positions p0 ..) of kv head hk, in
// page order: pages l_u, their device ids and the rows that chose them; returns
// their number.  What counts for nothing (negative, not yet visible, missing,
// repeated) is left out.  In page order, workgroups that run at the same time
// pass over the same pages at about the same time, while those are in L2.
//
// A table of one mask per page is filled and read back where it fits into the
// `cells` (even) 16-bit words at `table`, which hold nt * top ints at least; that costs
// a turn with two barriers per T pages.  A single row's ascending list of up to T
// entries (a decode step's) is taken as it is; otherwise every entry looks for its like
// among all (one row, pages of 16: 256 entries 16 us, 512 78, 1024 257).  The whole
// workgroup of T.
template <int T>
__device__ __forceinline__ int build_union(const SparseArgs& a, const SeqRows& s, int nt, int t0, int p0, int hk,
                                           uint32_t* table, int cells, int* l_u, int* l_id, uint16_t* l_mask, int* s_cnt) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int E = nt * a.top;
  auto entry = [&](int e, int* id) __attribute__((always_inline)) -> int {
    const int i = e / a.top, p = p0 + i;
    const int u = gptr(a.pages)[((size_t)(t0 + i) * a.hkv + hk) * a.top + e % a.top];
    *id = p < 0 || u > p / a.r.page ? -1 : page_id(a.r, s, u);
    return *id < 0 ? -1 : u;
  };
  // appends the workgroup's entries that are `own`, in thread order
  int nsel = 0;
  auto append = [&](bool own, int u, int mask, int id) __attribute__((always_inline)) {
    const uint64_t bal = __ballot(own);
    if (lane == 0) s_cnt[wave] = __popcll(bal);
    __syncthreads();
    int at = nsel + __popcll(bal & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < T / kWave; w++) {
      if (w < wave) at += s_cnt[w];
      nsel += s_cnt[w];
    }
    if (own) {
      l_u[at] = u;
      l_id[at] = id;
      l_mask[at] = (uint16_t)mask;
    }
    __syncthreads();
  };
  const int pmax = p0 + nt - 1, n = pmax < 0 ? 0 : min(pmax / a.r.page + 1, s.npg);
  if (nt > 1 && n <= cells) {
    for (int i = tid; i < (n + 1) / 2; i += T) table[i] = 0;
    __syncthreads();
    for (int e = tid; e < E; e += T) {
      int id;
      const int u = entry(e, &id);
      if (u >= 0) atomicOr(&table[u / 2], 1u << (e / a.top + 16 * (u % 2)));
    }
    __syncthreads();
    for (int u0 = 0; u0 < n; u0 += T) {
      const int u = u0 + tid, mask = u < n ? table[u / 2] >> (16 * (u % 2)) & 0xffff : 0;
      append(mask != 0, u, mask, mask ? page_id(a.r, s, u) : -1);
    }
  } else if (nt == 1 && E <= T) {  // a decode step's: an entry a thread
    int* const s_u = reinterpret_cast<int*>(table);
    int id = -1;
    const int u = tid < E ? entry(tid, &id) : -1;
    s_u[tid] = u;
    __syncthreads();
    bool own = u >= 0;
    if (__syncthreads_or(own && tid > 0 && (s_u[tid - 1] < 0 || u <= s_u[tid - 1])))  // not ascending: look for its like
      for (int j = 0; own && j < tid; j++) own = s_u[j] != u;
    append(own, u, 1, id);
  } else {
    int* const s_u = reinterpret_cast<int*>(table);
    int id;
    for (int e = tid; e < E; e += T) s_u[e] = entry(e, &id);
    __syncthreads();
    for (int e0 = 0; e0 < E; e0 += T) {
      const int e = e0 + tid, u = e < E ? s_u[e] : -1;
      bool own = u >= 0;
      int mask = 0;
      if (own)
        for (int j = 0; j < E; j++)
          if (s_u[j] == u) {
            mask |= 1 << (j / a.top);
            if (j < e) own = false;
          }
      append(own, u, mask, own ? page_id(a.r, s, u) : -1);
    }
  }
  return __builtin_amdgcn_readfirstlane(nsel);
}

// PG32: pages are a multiple of 32 tokens, so a block lies in one page
// and its address is uniform (else the lanes work out one token's each).
//
// K and V go straight into the wave's LDS slots; its next K block is requested
// as soon as this one's fragments are in registers and its next V block after
// P V, so one of the two is always in flight.
template <int DT, int D, bool PG32>
__global__ __launch_bounds__(SP_WAVES * kWave) void sparse_kernel(SparseArgs a) {
  constexpr int T = SP_WAVES * kWave;
  constexpr int RPI = 512 / D;      // rows per direct load (64 lanes of 16 bytes)
  constexpr int NL = SP_BLK / RPI;  // loads per operand of a block
  constexpr int CPR = D / 8;        // chunks per row
  __shared__ __attribute__((aligned(16))) uint16_t s_k[SP_WAVES][SP_BLK * D];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[SP_WAVES][SP_BLK * D];
  __shared__ int l_u[SP_MAX_ENTRIES], l_id[SP_MAX_ENTRIES];  // union: page, device page id, rows
  __shared__ uint16_t l_mask[SP_MAX_ENTRIES];
  __shared__ float s_m[SP_WAVES][16], s_l[SP_WAVES][16];
  __shared__ int s_cnt[SP_WAVES], s_tile[2];
  static_assert(SP_MAX_ENTRIES * 4 <= (int)sizeof(s_k), "the entries fit where K goes later");
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int split = blockIdx.x % a.splits, pair = blockIdx.x / a.splits;
  const int hk = pair % a.hkv, tile = pair / a.hkv;
  const int G = a.hq / a.hkv, col = lane % 16, grp = lane / 16;

  // ---- the tile's sequence and rows
  if (a.r.qo_indptr) {
    if (tid == 0) find_tile(a.r, tile, a.tt, s_tile);
    __syncthreads();
  }
  const int b = a.r.qo_indptr ? s_tile[0] : tile, i0 = a.r.qo_indptr ? s_tile[1] : 0;
  if (b >= a.r.batch) return;
  const SeqRows s = seq_rows(a.r, b);
  const int nt = min(a.tt, s.n - i0), t0 = s.row0 + i0, p0 = s.len - s.n + i0;  // rows, first row, its position
  const int pmax = p0 + nt - 1;

  // ---- this lane's query row: column col = row i of the tile, head g
  const int qi = col / G, qg = col % G;
  const bool qok = qi < nt;
  const int qpos = p0 + qi;
  uint4 qf[D / 32];
#pragma unroll
  for (int st = 0; st < D / 32; st++) {
    qf[st] = make_uint4(0, 0, 0, 0);
    if (qok) qf[st] = ldg16(a.q + ((size_t)(t0 + qi) * a.hq + (size_t)hk * G + qg) * D + 32 * st + 8 * grp);
  }

  const int nsel = build_union<T>(a, s, nt, t0, p0, hk, reinterpret_cast<uint32_t*>(&s_k[0][0]), (int)sizeof(s_k) / 2, l_u,
                                  l_id, l_mask, s_cnt);
  const int total = nsel * a.r.page;  // tokens of the union's pages
  const int nblk = (total + SP_BLK - 1) / SP_BLK;
  const int per = (nblk + a.splits - 1) / a.splits;
  const int blk0 = min(split * per, nblk), blk1 = min(blk0 + per, nblk);

  uint16_t* const ks = s_k[wave];
  uint16_t* const vs = s_v[wave];
  uint32_t koff[D / 32], voff[D / 16];
#pragma unroll
  for (int st = 0; st < D / 32; st++) koff[st] = col * D + 8 * ((4 * st + grp) ^ k_swz<D>(col));
  {
    const int r0 = 4 * grp + col / 4, qc = (col % 4) / 2, qh = 4 * (col % 2);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) voff[dt] = r0 * D + 8 * ((2 * dt + qc) ^ v_swz<D>(r0)) + qh;
  }
  const size_t tok_stride = (size_t)a.hkv * D;

  // Rows [j0, j1) of the tile at once.  Where the result is not finite, each row
  // again by itself with the values it does not see zeroed in LDS: infinity or
  // NaN in another row's token would reach it as 0 * inf through P V.
  int j0 = 0, j1 = nt;
  bool exact = false;
  while (true) {
    const int bits = ((1 << j1) - 1) & ~((1 << j0) - 1);
    // Tokens of a block: its first position, the rows that see its page and the
    // address of its first row (PG32), or those of token lane % 32.
    struct Block {
      int pos, mask;
      size_t off;
    };
    auto block = [&](int blk) __attribute__((always_inline)) -> Block {
      Block t;
      const int j = blk * SP_BLK + (PG32 ? 0 : lane % SP_BLK);
      const int e = min(j / a.r.page, nsel - 1), slot = j - e * a.r.page;  // (slot >= page behind the last page)
      int u = l_u[e], id = l_id[e], mask = l_mask[e];
      if constexpr (PG32) {
        u = __builtin_amdgcn_readfirstlane(u);
        id = __builtin_amdgcn_readfirstlane(id);
        mask = __builtin_amdgcn_readfirstlane(mask);
      }
      t.pos = u * a.r.page + slot;
      t.mask = j < total ? mask & bits : 0;
      // what no row of the tile sees yet is not read: the page's last visible token stands in
      const int at = PG32 ? slot : max(min(slot, min(pmax - u * a.r.page, a.r.page - 1)), 0);
      t.off = ((size_t)id * a.r.page + at) * tok_stride + (size_t)hk * D;
      return t;
    };
    auto issue = [&](const Block& t, auto is_k_c) __attribute__((always_inline)) {
      constexpr bool IS_K = decltype(is_k_c)::value;
      const uint16_t* const cache = IS_K ? a.kc : a.vc;
      uint16_t* const dst = IS_K ? ks : vs;
      auto rows = [&](auto whole_c) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NL; u++) {
          const int row = RPI * u + lane / CPR;
          const int chunk = 8 * ((lane % CPR) ^ (IS_K ? k_swz<D>(row) : v_swz<D>(row)));
          const uint16_t* src;
          if constexpr (decltype(whole_c)::value) {
            src = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(cache + t.off) +
                                                    2u * (uint32_t)(row * (int)tok_stride + chunk));
          } else if constexpr (PG32) {
            // rows that no row of the tile sees yet: the last visible one (in this page, maybe before the block)
            src = cache + t.off + (long long)min(row, pmax - t.pos) * (long long)tok_stride + chunk;
          } else {
            const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)t.off, row), hi = (uint32_t)__shfl((int)(t.off >> 32), row);
            src = cache + ((size_t)hi << 32 | lo) + chunk;
          }
          lds_load16(src, dst + RPI * u * D);
        }
      };
      if (PG32 && pmax - t.pos >= SP_BLK - 1) rows(std::true_type{});  // (uniform)
      else rows(std::false_type{});
    };
    float m_i = -INFINITY, l_i = 0.f;
    bool far = false;  // some row's m_i is beyond kFarScore
    f32x4 acc[D / 16];
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

    Block cur;
    // LAST: there is no next block (a copy of its own: every path knows how many loads are in flight)
    auto consume = [&](int blk, auto last_c) __attribute__((always_inline)) {
      constexpr bool LAST = decltype(last_c)::value;
      Block nxt;
      if constexpr (!LAST) nxt = block(blk + SP_WAVES);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");  // K has landed, V may be on its way
      f32x4 sc[2];
#pragma unroll
      for (int n = 0; n < 2; n++) {
        f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < D / 32; st++)
          c = mfma16<DT>(*reinterpret_cast<const uint4*>(&ks[koff[st] + 16 * n * D]), qf[st], c);
        sc[n] = c;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every K fragment is in registers
      if constexpr (!LAST) issue(nxt, std::true_type{});
      // mask: this lane's tokens are 16 n + 4 grp + i
      if constexpr (PG32) {
        const bool row = (cur.mask >> qi) & 1;
        if (cur.pos + SP_BLK - 1 <= p0 + j0) {  // (uniform) every row is behind the block
          if (cur.mask != bits) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
              for (int i = 0; i < 4; i++) sc[n][i] = row ? sc[n][i] : -INFINITY;
          }
        } else {
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              sc[n][i] = row && cur.pos + 16 * n + 4 * grp + i <= qpos ? sc[n][i] : -INFINITY;
        }
      } else if (__ballot(cur.mask != bits || cur.pos > p0 + j0)) {
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int mask = __shfl(cur.mask, 16 * n + 4 * grp + i), pos = __shfl(cur.pos, 16 * n + 4 * grp + i);
            sc[n][i] = ((mask >> qi) & 1) && pos <= qpos ? sc[n][i] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, sc[n][i]);
      mx = max_xor32(max_xor16(mx)) * a.scale_log2;
      if (__builtin_amdgcn_ballot_w64(mx > m_i + kLazy)) {
        const float mnew = mx > m_i + kLazy ? mx : m_i;
        const float alpha = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - mnew);
        m_i = mnew;
        far = __builtin_amdgcn_ballot_w64(fabsf(m_i) > kFarScore && m_i > -INFINITY) != 0;
        l_i *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) acc[dt] *= alpha;
      }
      float mref = m_i == -INFINITY ? 0.f : m_i, scale = a.scale_log2;
      if (far) {  // (uniform; a row goes by its own maximum, so its weights agree)
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) sc[n][i] = far_exponent(sc[n][i], scale, mref);
        mref = 0.f;
        scale = 1.f;
      }
      mref -= kPBias<DT>;
      float pv[2][4];
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          pv[n][i] = __builtin_amdgcn_exp2f(fmaf(sc[n][i], scale, -mref));
          l_i += pv[n][i];
        }
      const uint4 pb = make_uint4(pack2<DT>(pv[0][0], pv[0][1]), pack2<DT>(pv[0][2], pv[0][3]),
                                  pack2<DT>(pv[1][0], pv[1][1]), pack2<DT>(pv[1][2], pv[1][3]));
      if constexpr (!LAST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");  // V; the next K is on its way
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (exact) {
#pragma unroll
        for (int u = 0; u < NL; u++) {
          const int row = RPI * u + lane / CPR;
          const int mask = PG32 ? cur.mask : __shfl(cur.mask, row), pos = PG32 ? cur.pos + row : __shfl(cur.pos, row);
          if (!mask || pos > p0 + j0)
            *reinterpret_cast<uint4*>(vs + RPI * u * D + 8 * lane) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) {
        const uint2 lo = lds_tr4(&vs[voff[dt]]), hi = lds_tr4(&vs[voff[dt] + 16 * D]);
        acc[dt] = mfma16<DT>(make_uint4(lo.x, lo.y, hi.x, hi.y), pb, acc[dt]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every V fragment is in registers
      if constexpr (!LAST) {
        issue(nxt, std::false_type{});
        cur = nxt;
      }
    };
    // wave w takes blocks w, w + SP_WAVES, .. of the split (a fixed order)
    if (blk0 + wave < blk1) {
      int blk = blk0 + wave;
      cur = block(blk);
      issue(cur, std::true_type{});
      issue(cur, std::false_type{});
      for (; blk + SP_WAVES < blk1; blk += SP_WAVES) consume(blk, std::false_type{});
      consume(blk, std::true_type{});
    }

    // ---- the waves merge: O over each wave's own V slot
    l_i = add_xor32(add_xor16(l_i));
    float* const os = reinterpret_cast<float*>(vs);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) *reinterpret_cast<f32x4*>(os + col * D + 16 * dt + 4 * grp) = acc[dt];
    if (grp == 0) {
      s_m[wave][col] = m_i;
      s_l[wave][col] = l_i;
    }
    __syncthreads();
    const int live = min(SP_WAVES, blk1 - blk0);  // waves that had a block
    bool bad = false;
    for (int idx = tid; idx < 16 * D / 4; idx += T) {
      const int row = idx / (D / 4), d0 = idx % (D / 4) * 4, i = row / G, g = row % G;
      if (i < j0 || i >= j1) continue;
      float M = -INFINITY, L = 0.f;
      f32x4 O = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < live; w++) M = fmaxf(M, s_m[w][row]);
      for (int w = 0; w < live; w++) {
        const float f = s_m[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][row] - M);
        const f32x4 v = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(s_v[w]) + row * D + d0);
        L += s_l[w][row] * f;
        O += v * f;
      }
      const float sum = O[0] + O[1] + O[2] + O[3];
      bad |= !(fabsf(sum) < INFINITY);
      if (a.splits == 1) {
        const float inv = L > 0.f ? 1.f / L : 0.f;
        O *= inv;
        *reinterpret_cast<uint2*>(a.out + ((size_t)(t0 + i) * a.hq + (size_t)hk * G + g) * D + d0) =
            make_uint2(pack2<DT>(O[0], O[1]), pack2<DT>(O[2], O[3]));
      } else {
        float* rec = a.partial + (((size_t)pair * a.splits + split) * a.tt * G + row) * (D + 4);
        st_agent4(rec + d0, make_float4(O[0], O[1], O[2], O[3]));
        if (d0 == 0) st_agent4(rec + D, make_float4(M, L, 0.f, 0.f));
      }
    }
    const int again = __syncthreads_or(bad);
    if (!exact) {
      if (!again) break;
      exact = true;
      j0 = 0;
      j1 = 1;
    } else {
      if (j1 == nt) break;
      j0++;
      j1++;
    }
  }
  if (a.splits == 1) return;

  // ---- the splits meet in the workgroup that arrives last: a thread takes 4
  // dims of one row over every SG-th split, 8 records in flight, and the SG
  // parts meet in LDS (a fixed order)
  if (!arrive_last(&a.tickets[pair], a.splits)) return;
  constexpr int MU = 8;
  const int rows = nt * G, items = rows * (D / 4);
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
        if (d0 == 0) sml[j * 16 + row] = make_float2(M, L);
      }
      __syncthreads();
      if (!work || j > 0) return;
      float mb = -INFINITY;
      for (int u = 0; u < SG; u++) mb = fmaxf(mb, sml[u * 16 + row].x);
      L = 0.f;
      O = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int u = 0; u < SG; u++) {
        const float2 v = sml[u * 16 + row];
        const float f = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - mb);
        L += v.y * f;
        O += so[u * items + item] * f;
      }
    }
    if (work) {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      O *= inv;
      *reinterpret_cast<uint2*>(a.out + ((size_t)(t0 + row / G) * a.hq + (size_t)hk * G + row % G) * D + d0) =
          make_uint2(pack2<DT>(O[0], O[1]), pack2<DT>(O[2], O[3]));
    }
  }
}

// Many rows: four groups of 16 query rows (a wave each, the rows of up to
// 4 (16 / G) tokens) share one union.  Every 64-token block of it is loaded once
// by the whole workgroup, the next one while this one is worked on, and a wave
// skips the blocks that none of its rows chose.  Neighbouring rows choose much
// alike (777 rows of 16 pages: 36 pages for 4 rows, 65 for 16).  Bound by the slowest
// wave between two barriers: 1024 workgroups (2048 rows of 16 pages of 64, 8 kv heads
// of 4 heads of 128) take 207 us, MFMA busy for a tenth of it.
//
// Lane l of every wave knows token l of a block: its row in the cache and which
// rows of the tile see it.  A row's 64 tokens are then one ballot.
// PG64: pages are a multiple of 64 tokens, a block lies in one page and its
// address is uniform.
constexpr int SW_BLK = 64, SW_WAVES = 4;

template <int DT, int D, bool PG64>
__global__ __launch_bounds__(SW_WAVES * kWave, 2) void sparse_wide_kernel(SparseArgs a) {
  constexpr int T = SW_WAVES * kWave;
  constexpr int RPI = T * 8 / D;    // rows per load instruction of the workgroup
  constexpr int NL = SW_BLK / RPI;  // such loads per operand of a block
  constexpr int CPR = D / 8;        // chunks per row
  // separate objects: reads of one block do not wait for the loads that fill the other
  __shared__ __attribute__((aligned(16))) uint16_t s_k0[SW_BLK * D], s_k1[SW_BLK * D];
  __shared__ __attribute__((aligned(16))) uint16_t s_v0[SW_BLK * D], s_v1[SW_BLK * D];
  __shared__ int l_u[SP_MAX_ENTRIES], l_id[SP_MAX_ENTRIES];  // union: page, device page id, rows
  __shared__ uint16_t l_mask[SP_MAX_ENTRIES];
  __shared__ int s_cnt[SW_WAVES], s_tile[2], s_bad;
  static_assert(SP_MAX_ENTRIES * 4 <= (int)sizeof(s_k0), "the entries fit where K goes later");
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int hk = blockIdx.x % a.hkv, tile = blockIdx.x / a.hkv;
  const int G = a.hq / a.hkv, tb = 16 / G, col = lane % 16, grp = lane / 16;

  if (tid == 0) {
    find_tile(a.r, tile, a.tt, s_tile);
    s_bad = 0;
  }
  __syncthreads();
  const int b = s_tile[0], i0 = s_tile[1];
  if (b >= a.r.batch) return;
  const SeqRows s = seq_rows(a.r, b);
  const int nt = min(a.tt, s.n - i0), t0 = s.row0 + i0, p0 = s.len - s.n + i0;  // rows, first row, its position
  const int pmax = p0 + nt - 1;

  // ---- this lane's query row: column col = row qi of the tile, head qg
  const int qr = col / G, qi = wave * tb + qr, qg = col % G;
  const bool qok = qr < tb && qi < nt;
  uint4 qf[D / 32];
#pragma unroll
  for (int st = 0; st < D / 32; st++) {
    qf[st] = make_uint4(0, 0, 0, 0);
    if (qok) qf[st] = ldg16(a.q + ((size_t)(t0 + qi) * a.hq + (size_t)hk * G + qg) * D + 32 * st + 8 * grp);
  }
  const int nsel = build_union<T>(a, s, nt, t0, p0, hk, reinterpret_cast<uint32_t*>(s_k0), SW_BLK * D, l_u, l_id, l_mask,
                                  s_cnt);
  const int total = nsel * a.r.page, nblk = (total + SW_BLK - 1) / SW_BLK;
  const int step_e = SW_BLK / a.r.page, step_s = SW_BLK % a.r.page;  // entries and slots from block to block

  uint32_t koff[D / 32], voff[D / 16];
#pragma unroll
  for (int st = 0; st < D / 32; st++) koff[st] = col * D + 8 * ((4 * st + grp) ^ k_swz<D>(col));
  {
    const int r0 = 4 * grp + col / 4, qc = (col % 4) / 2, qh = 4 * (col % 2);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) voff[dt] = r0 * D + 8 * ((2 * dt + qc) ^ v_swz<D>(r0)) + qh;
  }
  const size_t tok_stride = (size_t)a.hkv * D;

  // Rows `bits` of the tile; exact: one row, with what it does not see zeroed (see sparse_kernel)
  auto pass = [&](int bits, bool exact) __attribute__((always_inline)) {
    const int mine = bits & (((1 << tb) - 1) << (wave * tb));  // this wave's rows
    float m_i = -INFINITY, l_i = 0.f;
    bool far = false;  // some row's m_i is beyond kFarScore
    f32x4 acc[D / 16];
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    int e = lane / a.r.page, slot = lane % a.r.page, at = lane;  // this lane's token of the block to load
    int vis = 0, vis_next = 0;  // rows that see this lane's token of the block at hand and of the next one
    size_t off = 0;
    int over = 0;  // (PG64) tokens of the block that some row of the tile sees, less one
    auto inform = [&]() __attribute__((always_inline)) {
      const int ec = min(e, nsel - 1);
      int u = l_u[ec], id = l_id[ec], mask = l_mask[ec];
      if constexpr (PG64) {
        u = __builtin_amdgcn_readfirstlane(u);
        id = __builtin_amdgcn_readfirstlane(id);
        const int slot0 = __builtin_amdgcn_readfirstlane(slot);
        over = pmax - (u * a.r.page + slot0);
        off = ((size_t)id * a.r.page + slot0) * tok_stride + (size_t)hk * D;
      } else {
        off = ((size_t)id * a.r.page + min(slot, pmax - u * a.r.page)) * tok_stride + (size_t)hk * D;
      }
      // rows at positions p0 + i >= this token's
      vis_next = at < total ? mask & bits & (-1 << min(max(u * a.r.page + slot - p0, 0), 16)) : 0;
      e += step_e;
      slot += step_s;
      if (slot >= a.r.page) {
        slot -= a.r.page;
        e++;
      }
      at += SW_BLK;
    };
    auto issue = [&](uint16_t* kd, uint16_t* vd) __attribute__((always_inline)) {
      auto rows = [&](auto whole_c) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NL; u++) {
          const int row = RPI * u + tid / CPR, c = lane % CPR;
          // a wave's part of the instruction: 512 / D rows from here on
          const int first = (RPI * u + wave * (512 / D)) * D, ck = 8 * (c ^ k_swz<D>(row)), cv = 8 * (c ^ v_swz<D>(row));
          if constexpr (decltype(whole_c)::value) {
            const uint32_t o = (uint32_t)row * (uint32_t)tok_stride;
            lds_load16(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(a.kc + off) + 2u * (o + ck)), kd + first);
            lds_load16(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(a.vc + off) + 2u * (o + cv)), vd + first);
          } else {
            size_t o;
            if constexpr (PG64) o = off + (long long)min(row, over) * (long long)tok_stride;  // (maybe before the block)
            else o = (size_t)(uint32_t)__shfl((int)(off >> 32), row) << 32 | (uint32_t)__shfl((int)(uint32_t)off, row);
            lds_load16(a.kc + o + ck, kd + first);
            lds_load16(a.vc + o + cv, vd + first);
          }
        }
      };
      if (PG64 && over >= SW_BLK - 1) rows(std::true_type{});  // (uniform)
      else rows(std::false_type{});
    };
    auto step = [&](int blk, const uint16_t* ks, uint16_t* vs, uint16_t* kn, uint16_t* vn) __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();  // the block has landed for every wave, and the one before is read out
      asm volatile("" ::: "memory");
      vis = vis_next;
      if (blk + 1 < nblk) {
        inform();
        issue(kn, vn);
      }
      if (exact) {  // (rare)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int u = 0; u < NL; u++)
          if (!__shfl(vis, RPI * u + tid / CPR)) *reinterpret_cast<uint4*>(vs + RPI * u * D + 8 * tid) = make_uint4(0, 0, 0, 0);
        __syncthreads();
      }
      if (!__ballot((vis & mine) != 0)) return;
      const bool whole = !__ballot((vis & mine) != mine);
      f32x4 sc[4];
#pragma unroll
      for (int n = 0; n < 4; n++) sc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < D / 32; st++)
#pragma unroll
        for (int n = 0; n < 4; n++)
          sc[n] = mfma16<DT>(*reinterpret_cast<const uint4*>(&ks[koff[st] + 16 * n * D]), qf[st], sc[n]);
      if (!whole) {
        uint64_t seen = 0;  // tokens that this lane's row sees
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint64_t row = __ballot((vis >> (wave * tb + i)) & 1);
          seen = qr == i ? row : seen;
        }
        const uint32_t lo = (uint32_t)seen >> (4 * grp), hi = (uint32_t)(seen >> 32) >> (4 * grp);
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) sc[n][i] = (n < 2 ? lo : hi) >> (16 * (n % 2) + i) & 1 ? sc[n][i] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 4; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, sc[n][i]);
      mx = max_xor32(max_xor16(mx)) * a.scale_log2;
      if (__builtin_amdgcn_ballot_w64(mx > m_i + kLazy)) {
        const float mnew = mx > m_i + kLazy ? mx : m_i;
        const float alpha = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - mnew);
        m_i = mnew;
        far = __builtin_amdgcn_ballot_w64(fabsf(m_i) > kFarScore && m_i > -INFINITY) != 0;
        l_i *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) acc[dt] *= alpha;
      }
      float mref = m_i == -INFINITY ? 0.f : m_i, scale = a.scale_log2;
      if (far) {  // (uniform; a row goes by its own maximum, so its weights agree)
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) sc[n][i] = far_exponent(sc[n][i], scale, mref);
        mref = 0.f;
        scale = 1.f;
      }
      mref -= kPBias<DT>;
      uint4 pb[2];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        float pv[2][4];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            pv[n][i] = __builtin_amdgcn_exp2f(fmaf(sc[2 * m + n][i], scale, -mref));
            l_i += pv[n][i];
          }
        pb[m] = make_uint4(pack2<DT>(pv[0][0], pv[0][1]), pack2<DT>(pv[0][2], pv[0][3]), pack2<DT>(pv[1][0], pv[1][1]),
                           pack2<DT>(pv[1][2], pv[1][3]));
      }
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) {
          const uint2 lo = lds_tr4(&vs[voff[dt] + 32 * m * D]), hi = lds_tr4(&vs[voff[dt] + (32 * m + 16) * D]);
          acc[dt] = mfma16<DT>(make_uint4(lo.x, lo.y, hi.x, hi.y), pb[m], acc[dt]);
        }
    };
    if (nblk > 0) {
      inform();
      issue(s_k0, s_v0);
    }
    for (int blk = 0; blk < nblk; blk += 2) {
      step(blk, s_k0, s_v0, s_k1, s_v1);
      if (blk + 1 < nblk) step(blk + 1, s_k1, s_v1, s_k0, s_v0);
    }
    l_i = add_xor32(add_xor16(l_i));
    const float inv = l_i > 0.f ? 1.f / l_i : 0.f;
    float sum = 0.f;
    if (qok && (mine >> qi & 1)) {
      uint16_t* const o = a.out + ((size_t)(t0 + qi) * a.hq + (size_t)hk * G + qg) * D + 4 * grp;
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) {
        const f32x4 v = acc[dt] * inv;
        sum += v[0] + v[1] + v[2] + v[3];
        *reinterpret_cast<uint2*>(o + 16 * dt) = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
      }
    }
    if (!exact && !(fabsf(sum) < INFINITY)) atomicOr(&s_bad, 1 << qi);
    __syncthreads();  // the blocks' slots are free again
  };
  pass((1 << nt) - 1, false);
  for (int bad = s_bad; bad; bad &= bad - 1) pass(bad & -bad, true);
}

// Tiles, rows per tile and splits of a call.
struct SparsePlan {
  long long tiles;
  int tt, splits;
  bool wide;
};
static SparsePlan sparse_plan(bool ragged, int rows, int batch, int hkv, int G, int page, int top) {
  SparsePlan p;
  // Four groups of rows to a tile where its workgroups, two a CU, fill their rounds
  // well enough and the lists fit.  One group to a tile loads shared pages again, in
  // any number of workgroups, and works out every token's address unless pages are a
  // multiple of 32 (8 kv heads of 4, d = 128; rows, pages, us with four groups and one):
  // 256 16 of 64 98 37; 777 16 of 64 120 107; 777 16 of 16 53 74; 1200 16 of 64 177 141;
  // 2048 16 of 64 207 219, 64 of 16 260 394, 32 of 32 255 225; 2048 of 8 heads, d = 64, 161
  // 167.  Rows of many sequences, whose last tiles are not full, come out alike: up to 4
  // rows in each of 256, 16 of 64 316 357, 16 of 16 153 206.
  const int wide_tt = SW_WAVES * (16 / G);
  const long long wide = ((long long)rows + wide_tt - 1) / wide_tt * hkv, slots = (wide + 511) / 512 * 512;
  p.wide = ragged && G >= 4 && wide_tt * top <= SP_MAX_ENTRIES && 100 * slots < wide * (page % SP_BLK ? 140 : 108);
  if (p.wide) {
    p.tt = wide_tt;
    p.tiles = (long long)rows / p.tt + batch;
    if (p.tiles > rows) p.tiles = rows;
    p.splits = 1;
    return p;
  }
  p.tt = ragged ? 16 / G : 1;
  if (p.tt > SP_MAX_ENTRIES / top) p.tt = SP_MAX_ENTRIES / top;
  p.tiles = ragged ? (long long)rows / p.tt + batch : rows;
  if (p.tiles > rows) p.tiles = rows;
  const long long pairs = p.tiles * hkv, blocks = ((long long)p.tt * top * page + SP_BLK - 1) / SP_BLK;
  long long sp = SP_TARGET_WG / pairs;
  if (sp > blocks / SP_MIN_BLOCKS) sp = blocks / SP_MIN_BLOCKS;
  if (pairs > kMaxTickets || sp < 1) sp = 1;
  p.splits = (int)sp;
  return p;
}

}  // namespace yr

using namespace yr;

extern "C" size_t yr_hip_gqa_sparse_workspace(int rows, int batch, int ragged, int hq, int hkv, int d, int page_size,
                                              int top_pages) {
  if (rows <= 0 || batch <= 0 || hkv <= 0 || hq < hkv || hq % hkv || hq / hkv > 16 || page_size <= 0 || top_pages < 1 ||
      top_pages > SP_MAX_ENTRIES || d <= 0)
    return 0;
  const SparsePlan p = sparse_plan(ragged != 0, rows, batch, hkv, hq / hkv, page_size, top_pages);
  if (p.splits == 1) return 0;
  return kTicketBytes + (size_t)p.tiles * hkv * p.splits * p.tt * (hq / hkv) * (d + 4) * sizeof(float);
}

extern "C" int yr_hip_gqa_sparse_plan(int rows, int batch, int ragged, int hq, int hkv, int page_size, int top_pages, int* plan3) {
  const char* nm = "yr_hip_gqa_sparse_plan";
  if (!plan3 || rows <= 0 || batch <= 0 || hkv <= 0 || hq < hkv || hq % hkv || hq / hkv > 16 || page_size <= 0 ||
      top_pages < 1 || top_pages > SP_MAX_ENTRIES)
    return fail(YR_E_INVALID, "%s: shape", nm);
  const SparsePlan p = sparse_plan(ragged != 0, rows, batch, hkv, hq / hkv, page_size, top_pages);
  plan3[0] = p.tt;
  plan3[1] = p.wide;
  plan3[2] = p.splits;
  return YR_OK;
}

extern "C" int yr_hip_gqa_sparse_paged(const void* q, const void* k_cache, const void* v_cache,
                                       const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                                       int n_indices, const int32_t* kv_len, const int32_t* pages, void* out, int rows,
                                       int batch, int hq, int hkv, int d, int page_size, int num_pages, int top_pages,
                                       int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* nm = "yr_hip_gqa_sparse_paged";
  SparseArgs a;
  a.r = Ragged{qo_indptr, kv_indptr, kv_indices, kv_len, rows, batch, page_size, n_indices, num_pages};
  if (!q || !k_cache || !v_cache || !pages || !out) return fail(YR_E_INVALID, "%s: null pointer", nm);
  int rc = ragged_check(nm, a.r, hq, hkv, d, dtype);
  if (rc != YR_OK) return rc;
  const int G = hq / hkv;
  if (G < 1 || G > 16) return fail(YR_E_INVALID, "%s: group size %d (1 to 16)", nm, G);
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15)
    return fail(YR_E_INVALID, "%s: pointers must be 16-byte aligned", nm);
  if (top_pages < 1 || top_pages > SP_MAX_ENTRIES)
    return fail(YR_E_INVALID, "%s: top_pages %d (1 to %d)", nm, top_pages, SP_MAX_ENTRIES);
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.pages = pages;
  a.out = (uint16_t*)out;
  a.hq = hq;
  a.hkv = hkv;
  a.top = top_pages;
  const SparsePlan p = sparse_plan(qo_indptr != nullptr, rows, batch, hkv, G, page_size, top_pages);
  a.tt = p.tt;
  a.splits = p.splits;
  if ((long long)p.tt * top_pages * page_size > 0x7fffffff)
    return fail(YR_E_INVALID, "%s: %d pages of %d tokens a row are too many", nm, top_pages, page_size);
  if ((long long)rows * hkv > 0x7fffffff || p.tiles * hkv * p.splits > 0x7fffffff)
    return fail(YR_E_INVALID, "%s: too many rows", nm);
  if ((long long)hkv * d * 2 * SP_BLK > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many heads", nm);
  const size_t need = yr_hip_gqa_sparse_workspace(rows, batch, qo_indptr != nullptr, hq, hkv, d, page_size, top_pages);
  if (need > workspace_bytes || (need && !workspace))
    return fail(YR_E_WORKSPACE, "%s: workspace %zu < %zu", nm, workspace_bytes, need);
  a.tickets = (uint32_t*)workspace;
  a.partial = need ? (float*)((char*)workspace + kTicketBytes) : nullptr;
  a.scale_log2 = kLog2e / sqrtf((float)d);
  const unsigned grid = (unsigned)(p.tiles * hkv * p.splits);
  const bool pg32 = page_size % SP_BLK == 0 && !p.wide;
  hipStream_t st = (hipStream_t)stream;
#define YR_SP(DT_, D_, P_)                                                                                  \
  if (dtype == DT_ && d == D_ && !p.wide && pg32 == P_)                                                     \
    hipLaunchKernelGGL((sparse_kernel<DT_, D_, P_>), dim3(grid), dim3(SP_WAVES * kWave), 0, st, a);
#define YR_SP2(DT_, D_)                                                                                     \
  if (dtype == DT_ && d == D_ && p.wide && page_size % SW_BLK == 0)                                         \
    hipLaunchKernelGGL((sparse_wide_kernel<DT_, D_, true>), dim3(grid), dim3(SW_WAVES * kWave), 0, st, a);  \
  if (dtype == DT_ && d == D_ && p.wide && page_size % SW_BLK != 0)                                         \
    hipLaunchKernelGGL((sparse_wide_kernel<DT_, D_, false>), dim3(grid), dim3(SW_WAVES * kWave), 0, st, a); \
  YR_SP(DT_, D_, false) YR_SP(DT_, D_, true)
  YR_SP2(DT_F16, 64) YR_SP2(DT_F16, 128) YR_SP2(DT_BF16, 64) YR_SP2(DT_BF16, 128)
#undef YR_SP2
#undef YR_SP
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
