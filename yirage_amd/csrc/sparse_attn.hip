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
#include "attn_device.h"
#include "ragged.h"

namespace yr {

constexpr int SP_WAVES = 8;
constexpr int SP_THREADS = SP_WAVES * kWave;
constexpr int SP_BLK = 32;           // tokens per wave block
constexpr int SP_MAX_ENTRIES = 1024; // list entries of a tile

struct SparseArgs {
  Ragged r;
  const uint16_t* q;      // [rows][hq][D]
  const uint16_t* kc;     // [pages][page][hkv][D]
  const uint16_t* vc;
  const int32_t* pages;   // [rows][hkv][top]
  uint16_t* out;
  int hq, hkv, top, tt, tiles;  // tt: rows per tile
  float scale_log2;
};

// P is stored in 16 bits for the second product.  f16's normal range ends at
// 2^-14: weights carry a factor 2^7 there (cancelled by the row sum, at most
// 2^15 with the lazy maximum's slack of 2^8), so a weight loses bits only below
// 2^-21 of the largest and vanishes below 2^-32.
template <int DT>
constexpr float kPBias = DT == DT_F16 ? 7.f : 0.f;

// 16-byte chunk permutations of an LDS row of D elements.  K fragments read one
// chunk column of 16 consecutive rows, transposing V reads a chunk pair of 4
// consecutive rows: any 8 lanes of either hit 8 chunks apart modulo 128 bytes.
template <int D>
__device__ __forceinline__ int k_swz(int row) { return row & (D == 128 ? 15 : 7); }
template <int D>
__device__ __forceinline__ int v_swz(int row) {
  return D == 128 ? ((row & 7) << 1) | ((row >> 3) & 1) : (row & 3) << 1;
}

template <int DT, int D>
__global__ __launch_bounds__(SP_THREADS) void sparse_kernel(SparseArgs a) {
  constexpr int RPI = 512 / D;         // rows per direct load (64 lanes of 16 bytes)
  constexpr int NL = SP_BLK / RPI;     // loads per operand of a block
  constexpr int CPR = D / 8;           // chunks per row
  __shared__ __attribute__((aligned(16))) uint16_t s_k[SP_WAVES][SP_BLK * D];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[SP_WAVES][SP_BLK * D];
  __shared__ float s_m[SP_WAVES][16], s_l[SP_WAVES][16];
  __shared__ int s_cnt[SP_WAVES], s_tile[3];
  __shared__ int s_u[SP_MAX_ENTRIES];  // page of each entry, -1: counts for nothing
  __shared__ int l_u[SP_MAX_ENTRIES], l_id[SP_MAX_ENTRIES], l_mask[SP_MAX_ENTRIES];  // union: page, device page id, rows
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int hk = blockIdx.x % a.hkv, tile = blockIdx.x / a.hkv;
  const int G = a.hq / a.hkv, col = lane % 16, grp = lane / 16;

  // ---- the tile's sequence and rows
  if (tid == 0) find_tile(a.r, tile, a.tt, s_tile);
  __syncthreads();
  const int b = s_tile[0], i0 = s_tile[1];
  if (b >= a.r.batch) return;
  const SeqRows s = seq_rows(a.r, b);
  const int nt = min(a.tt, s.n - i0), t0 = s.row0 + i0, p0 = s.len - s.n + i0;  // rows, first row, its position
  const int pmax = p0 + nt - 1;

  // ---- union of the rows' lists
  const int E = nt * a.top;
  for (int e = tid; e < E; e += SP_THREADS) {
    const int i = e / a.top, p = p0 + i;
    int u = gptr(a.pages)[((size_t)(t0 + i) * a.hkv + hk) * a.top + e % a.top];
    if (u < 0 || p < 0 || u > p / a.r.page || page_id(a.r, s, u) < 0) u = -1;
    s_u[e] = u;
  }
  __syncthreads();
  int nsel = 0;
  for (int e0 = 0; e0 < E; e0 += SP_THREADS) {
    const int e = e0 + tid;
    const int u = e < E ? s_u[e] : -1;
    bool own = u >= 0;
    int mask = 0;
    if (own)
      for (int i = 0; i < nt; i++)
        for (int j = 0; j < a.top; j++)
          if (s_u[i * a.top + j] == u) {
            mask |= 1 << i;
            if (i * a.top + j < e) own = false;
          }
    const uint64_t bal = __ballot(own);
    if (lane == 0) s_cnt[wave] = __popcll(bal);
    __syncthreads();
    int at = nsel + __popcll(bal & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < SP_WAVES; w++) {
      if (w < wave) at += s_cnt[w];
      nsel += s_cnt[w];
    }
    if (own) {
      l_u[at] = u;
      l_id[at] = page_id(a.r, s, u);
      l_mask[at] = mask;
    }
    __syncthreads();
  }
  const int total = nsel * a.r.page;  // tokens of the union's pages
  const int nblk = (total + SP_BLK - 1) / SP_BLK;

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
    const int plim = p0 + j1 - 1, bits = ((1 << j1) - 1) & ~((1 << j0) - 1);
    // element offset of virtual token j's row (of one that may be read where j is none)
    auto row_of = [&](int j) __attribute__((always_inline)) -> size_t {
      const int e = min(j / a.r.page, nsel - 1);
      const int slot = max(min(j < total ? j % a.r.page : 0, pmax - l_u[e] * a.r.page), 0);
      return ((size_t)l_id[e] * a.r.page + slot) * tok_stride + (size_t)hk * D;
    };
    auto issue = [&](int blk, auto is_k_c) __attribute__((always_inline)) {
      constexpr bool IS_K = decltype(is_k_c)::value;
      const uint16_t* cache = IS_K ? a.kc : a.vc;
      uint16_t* dst = IS_K ? ks : vs;
#pragma unroll
      for (int u = 0; u < NL; u++) {
        const int row = RPI * u + lane / CPR;
        const int chunk = (lane % CPR) ^ (IS_K ? k_swz<D>(row) : v_swz<D>(row));
        lds_load16(cache + row_of(blk * SP_BLK + row) + 8 * chunk, dst + RPI * u * D);
      }
    };
    float m_i = -INFINITY, l_i = 0.f;
    f32x4 acc[D / 16];
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int blk = wave; blk < nblk; blk += SP_WAVES) {
      issue(blk, std::true_type{});
      issue(blk, std::false_type{});
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (exact) {
#pragma unroll
        for (int u = 0; u < NL; u++) {
          const int j = blk * SP_BLK + RPI * u + lane / CPR, e = min(j / a.r.page, nsel - 1);
          const bool see = j < total && (l_mask[e] & bits) && l_u[e] * a.r.page + j % a.r.page <= plim;
          if (!see) *reinterpret_cast<uint4*>(vs + RPI * u * D + 8 * lane) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      f32x4 sc[2];
#pragma unroll
      for (int n = 0; n < 2; n++) {
        f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < D / 32; st++)
          c = mfma16<DT>(*reinterpret_cast<const uint4*>(&ks[koff[st] + 16 * n * D]), qf[st], c);
        sc[n] = c;
      }
      // mask: tokens 16 n + 4 grp + i of the block
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int j = blk * SP_BLK + 16 * n + 4 * grp + i, e = min(j / a.r.page, nsel - 1);
          const bool see = j < total && qok && qi >= j0 && qi < j1 && ((l_mask[e] >> qi) & 1) &&
                           l_u[e] * a.r.page + j % a.r.page <= qpos;
          sc[n][i] = see ? sc[n][i] : -INFINITY;
          mx = fmaxf(mx, sc[n][i]);
        }
      mx = max_xor32(max_xor16(mx)) * a.scale_log2;
      if (__builtin_amdgcn_ballot_w64(mx > m_i + kLazy)) {
        const float mnew = mx > m_i + kLazy ? mx : m_i;
        const float alpha = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - mnew);
        m_i = mnew;
        l_i *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) acc[dt] *= alpha;
      }
      const float mref = (m_i == -INFINITY ? 0.f : m_i) - kPBias<DT>;
      float pv[2][4];
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          pv[n][i] = __builtin_amdgcn_exp2f(fmaf(sc[n][i], a.scale_log2, -mref));
          l_i += pv[n][i];
        }
      const uint4 pb = make_uint4(pack2<DT>(pv[0][0], pv[0][1]), pack2<DT>(pv[0][2], pv[0][3]),
                                  pack2<DT>(pv[1][0], pv[1][1]), pack2<DT>(pv[1][2], pv[1][3]));
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) {
        const uint2 lo = lds_tr4(&vs[voff[dt]]), hi = lds_tr4(&vs[voff[dt] + 16 * D]);
        acc[dt] = mfma16<DT>(make_uint4(lo.x, lo.y, hi.x, hi.y), pb, acc[dt]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every fragment is in registers
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
    bool bad = false;
    for (int idx = tid; idx < 16 * D / 4; idx += SP_THREADS) {
      const int row = idx / (D / 4), d0 = idx % (D / 4) * 4, i = row / G, g = row % G;
      if (i < j0 || i >= j1) continue;
      float M = -INFINITY, L = 0.f;
      f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < SP_WAVES; w++) M = fmaxf(M, s_m[w][row]);
#pragma unroll
      for (int w = 0; w < SP_WAVES; w++) {
        const float f = s_m[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][row] - M);
        const f32x4 v = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(s_v[w]) + row * D + d0);
        L += s_l[w][row] * f;
        O += v * f;
      }
      const float inv = L > 0.f ? 1.f / L : 0.f;
      O *= inv;
      const float sum = O[0] + O[1] + O[2] + O[3];
      bad |= !(fabsf(sum) < INFINITY);
      *reinterpret_cast<uint2*>(a.out + ((size_t)(t0 + i) * a.hq + (size_t)hk * G + g) * D + d0) =
          make_uint2(pack2<DT>(O[0], O[1]), pack2<DT>(O[2], O[3]));
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
}

}  // namespace yr

using namespace yr;

extern "C" int yr_hip_gqa_sparse_paged(const void* q, const void* k_cache, const void* v_cache,
                                       const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                                       int n_indices, const int32_t* kv_len, const int32_t* pages, void* out, int rows,
                                       int batch, int hq, int hkv, int d, int page_size, int num_pages, int top_pages,
                                       int dtype, void* stream) {
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
  a.tt = qo_indptr ? 16 / G : 1;
  if (a.tt > SP_MAX_ENTRIES / top_pages) a.tt = SP_MAX_ENTRIES / top_pages;
  if ((long long)a.tt * top_pages * page_size > 0x7fffffff)
    return fail(YR_E_INVALID, "%s: %d pages of %d tokens a row are too many", nm, top_pages, page_size);
  a.scale_log2 = kLog2e / sqrtf((float)d);
  long long tiles = qo_indptr ? (long long)rows / a.tt + batch : rows;
  if (tiles > rows) tiles = rows;
  if (tiles * hkv > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
  a.tiles = (int)tiles;
  hipStream_t st = (hipStream_t)stream;
#define YR_SP(DT_, D_)                                                                                             \
  if (dtype == DT_ && d == D_)                                                                                     \
    hipLaunchKernelGGL((sparse_kernel<DT_, D_>), dim3((unsigned)(tiles * hkv)), dim3(SP_THREADS), 0, st, a);
  YR_SP(DT_F16, 64) YR_SP(DT_F16, 128) YR_SP(DT_BF16, 64) YR_SP(DT_BF16, 128)
#undef YR_SP
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
