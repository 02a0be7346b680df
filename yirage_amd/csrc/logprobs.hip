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
// The top costs one comparison a tile: a wave compares the lanes' tile maxima
// (formed for m anyway) with the worst key that can still be among its top, and
// looks at single elements only where one beats it.  That bound starts as the
// top-th largest of 64 lane maxima and moves whenever the wave's buffer of
// candidates is reduced.  Keys order by value, then by the lower index, so the
// result does not depend on the order in which candidates are found.
//
// NaN values take no part in the top (as in argmax) and make the sums NaN; a
// row of nothing but -inf has no distribution: NaN too.  A token outside
// [0, n_valid) has log probability NaN.
#include "yr_common.h"

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
constexpr int LP_TARGET_WG = 1024;

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
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int l) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}

// How many of the 64 lanes' keys beat this lane's.
__device__ __forceinline__ int wave_rank(uint64_t k) {
  int r = 0;
#pragma unroll 8
  for (int l = 0; l < kWave; l++) r += lane_u64(k, l) > k;
  return r;
}

// The `top` best of a wave's `count` keys in `buf`, in order, written back to
// buf[0, top) (0 where there are fewer).  Keys differ from one another.
__device__ __forceinline__ void wave_top(uint64_t* buf, int count, int top) {
  const int lane = threadIdx.x % kWave;
  if (count <= kWave) {
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

// Joins of (m, s, t): s and t relative to m (m = -inf: nothing yet, s = t = 0).
__device__ __forceinline__ void lp_rescale(double& s, double& t, float from, float to) {
  if (from == to) return;
  if (from == -INFINITY) return;  // s = t = 0 (or NaN, which stays)
  const double d = (double)from - (double)to, f = __expf((float)d);
  t = f == 0 ? 0 * t : f * (t + d * s);
  s *= f;
}

__device__ __forceinline__ void st_u64(uint64_t* p, uint64_t v) {
  __hip_atomic_store((YR_G uint64_t*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t ld_u64(const uint64_t* p) {
  return __hip_atomic_load((const YR_G uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int DT>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(LogprobArgs a) {
  constexpr int EPP = DT == YR_DTYPE_F32 ? 4 : 8;  // elements per 16-byte piece
  constexpr int U = 32 / EPP;                      // pieces per lane and tile
  constexpr int ES = 16 / EPP;
  __shared__ uint64_t s_buf[LP_WAVES][LP_BUF];
  extern __shared__ uint64_t s_list[];  // [splits][top]
  __shared__ float s_m[LP_WAVES];
  __shared__ double s_s[LP_WAVES], s_t[LP_WAVES];
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const char* x = (const char*)a.x + (size_t)row * a.stride * ES;
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
  uint64_t* const buf = s_buf[wave];
  float m = -INFINITY, bound = -INFINITY;  // bound: value of the worst key still wanted
  uint64_t worst = 0;                      // keys above it are still wanted
  int count = 0;
  double s = 0, t = 0;
  for (int p0 = p_begin + wave * (kWave * U); p0 < p_end; p0 += LP_WAVES * kWave * U) {
    float v[U][EPP];
    const bool inside = p0 > 0 && (p0 + kWave * U) * EPP - lead <= a.n && p0 + kWave * U <= p_end;  // uniform
    if (inside || (lead == 0 && (p0 + kWave * U) * EPP <= a.n && p0 + kWave * U <= p_end)) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; u++) w[u] = ldg16(x + ((long long)(p0 + u * kWave + lane) * EPP - lead) * ES);
#pragma unroll
      for (int u = 0; u < U; u++) {
        if constexpr (DT == YR_DTYPE_F32) {
          v[u][0] = __uint_as_float(w[u].x); v[u][1] = __uint_as_float(w[u].y);
          v[u][2] = __uint_as_float(w[u].z); v[u][3] = __uint_as_float(w[u].w);
        } else {
          v[u][0] = lo16<DT>(w[u].x); v[u][1] = hi16<DT>(w[u].x); v[u][2] = lo16<DT>(w[u].y); v[u][3] = hi16<DT>(w[u].y);
          v[u][4] = lo16<DT>(w[u].z); v[u][5] = hi16<DT>(w[u].z); v[u][6] = lo16<DT>(w[u].w); v[u][7] = hi16<DT>(w[u].w);
        }
      }
    } else {  // -inf stands for what is not there; it adds nothing and is told apart by its index below
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int p = p0 + u * kWave + lane;
#pragma unroll
        for (int e = 0; e < EPP; e++) {
          const int i = p * EPP - lead + e;
          v[u][e] = p < p_end && i >= 0 && i < a.n ? at(i) : -INFINITY;
        }
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < EPP; e++) mx = fmaxf(mx, v[u][e]);
    if (__ballot(mx > m)) {
      const float to = wave_maxf(fmaxf(mx, m));
      lp_rescale(s, t, m, to);
      m = to;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float st = 0.f, tt = 0.f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      float es = 0.f;
#pragma unroll
      for (int e = 0; e < EPP; e++) {
        const float y = v[u][e] - ref, ex = __expf(y);
        es += ex;
        tt = fmaf(ex, fmaxf(y, -1e4f), tt);  // (0 * -inf is none)
      }
      st += es;
    }
    s += st;
    t += tt;

    if (a.top > 0 && __ballot(mx >= bound)) {
      // the elements' keys; 0: no element, NaN or not above `worst`
      auto key_of = [&](int u, int e) __attribute__((always_inline)) -> uint64_t {
        const int p = p0 + u * kWave + lane, i = p * EPP - lead + e;
        const float f = v[u][e];
        return p < p_end && i >= 0 && i < a.n && f == f ? lp_key(f, i) : 0;
      };
      if (worst == 0 || __popcll(__ballot(mx >= bound)) > 16) {
        uint64_t k = 0;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int e = 0; e < EPP; e++) {
            const uint64_t c = key_of(u, e);
            k = c > k ? c : k;
          }
        // `top` keys at least are as good as the top-th best lane's: keep it and what beats it
        const int r = wave_rank(k);
        const uint64_t hit = __ballot(k != 0 && r == a.top - 1);
        if (hit) {
          const uint64_t b = lane_u64(k, __builtin_ctzll(hit)) - 1;
          if (b > worst) worst = b;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < EPP; e++) {
          uint64_t k = key_of(u, e);
          uint64_t take = __ballot(k > worst);
          if (take) {
            if (count + __popcll(take) > LP_BUF) {
              wave_top(buf, count, a.top);
              count = a.top;  // (the buffer was fuller than top)
              const uint64_t b = buf[a.top - 1];
              if (b > worst) worst = b;
              take = __ballot(k > worst);
            }
            if (k > worst) buf[count + __popcll(take & ((1ull << lane) - 1))] = k;
            count += __popcll(take);
          }
        }
      bound = worst ? lp_value(worst) : -INFINITY;  // (one below a key: the same value, the next index)
    }
  }
  if (a.top > 0) wave_top(buf, count, a.top);
  s = wave_sum_d(s);
  t = wave_sum_d(t);
  if (lane == 0) {
    s_m[wave] = m;
    s_s[wave] = s;
    s_t[wave] = t;
  }
  __syncthreads();
  // ---- the waves' numbers and lists
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < LP_WAVES; w++) M = fmaxf(M, s_m[w]);
  s = t = 0;
#pragma unroll
  for (int w = 0; w < LP_WAVES; w++) {
    double sw = s_s[w], tw = s_t[w];
    lp_rescale(sw, tw, s_m[w], M);
    s += sw;
    t += tw;
  }
  // position of a key in the joined list: how many of every wave's keys beat it
  for (int i = tid; i < a.top; i += LP_THREADS) s_list[i] = 0;
  __syncthreads();
  for (int i = tid; i < LP_WAVES * a.top; i += LP_THREADS) {
    const uint64_t k = s_buf[i / a.top][i % a.top];
    int r = 0;
    for (int q = 0; q < a.top; q++)
#pragma unroll
      for (int w = 0; w < LP_WAVES; w++) r += s_buf[w][q] > k;
    if (k && r < a.top) s_list[r] = k;
  }
  __syncthreads();

  if (a.splits > 1) {
    const int rec_len = 3 + a.top;
    uint64_t* rec = a.records + (size_t)row * a.splits * rec_len;
    if (tid == 0) {
      st_u64(rec + (size_t)split * rec_len, (uint64_t)__double_as_longlong((double)M));
      st_u64(rec + (size_t)split * rec_len + 1, (uint64_t)__double_as_longlong(s));
      st_u64(rec + (size_t)split * rec_len + 2, (uint64_t)__double_as_longlong(t));
    }
    for (int i = tid; i < a.top; i += LP_THREADS) st_u64(rec + (size_t)split * rec_len + 3 + i, s_list[i]);
    if (!arrive_last(&a.tickets[row], a.splits)) return;
    for (int i = tid; i < a.splits * a.top; i += LP_THREADS)
      s_list[i] = ld_u64(rec + (size_t)(i / a.top) * rec_len + 3 + i % a.top);
    __syncthreads();
    if (wave != 0) return;
    double ms = -INFINITY, ss = 0, ts = 0;
    if (lane < a.splits) {
      ms = __longlong_as_double((long long)ld_u64(rec + (size_t)lane * rec_len));
      ss = __longlong_as_double((long long)ld_u64(rec + (size_t)lane * rec_len + 1));
      ts = __longlong_as_double((long long)ld_u64(rec + (size_t)lane * rec_len + 2));
    }
    M = wave_maxf((float)ms);
    lp_rescale(ss, ts, (float)ms, M);
    s = wave_sum_d(ss);
    t = wave_sum_d(ts);
    // the splits' ordered lists: take the best head, `top` times
    int next = 0;
    uint64_t head = lane < a.splits && a.top > 0 ? s_list[lane * a.top] : 0, mine = 0;
    for (int k = 0; k < a.top; k++) {
      const uint64_t best = wave_max_key(head);
      if (lane == k) mine = best;
      if (best && head == best) {
        next++;
        head = next < a.top ? s_list[lane * a.top + next] : 0;
      }
    }
    if (lane < a.top) s_list[lane] = mine;  // (every head was read: the wave runs in step)
  }
  if (M == -INFINITY) s = t = NAN;  // no value at all
  const double ls = log(s);
  if (tid == 0) {
    gptr(a.logprob)[row] = (float)((double)(given - M) - ls);
    gptr(a.entropy)[row] = (float)(ls - t / s);
  }
  if (tid < a.top) {
    const uint64_t k = s_list[tid];
    gptr(a.top_lp)[(size_t)row * a.top + tid] = k ? (float)((double)(lp_value(k) - M) - ls) : -INFINITY;
    gptr(a.top_ids)[(size_t)row * a.top + tid] = k ? lp_index(k) : -1;
  }
}

// A row is split until about LP_TARGET_WG workgroups run, each with one tile of
// all its waves at least.
static void logprobs_plan(int rows, int n, int dtype, int* splits, int* chunk) {
  const int epp = dtype == YR_DTYPE_F32 ? 4 : 8, tile = LP_THREADS * 32 / epp;  // pieces
  const int np = (n - 1) / epp + 2;  // a row off its boundary has one more
  int sp = (LP_TARGET_WG + rows - 1) / rows;
  if (sp > LP_MAX_SPLITS) sp = LP_MAX_SPLITS;
  const int most = (np + tile - 1) / tile;
  if (sp > most) sp = most;
  *chunk = ((np + sp - 1) / sp + tile - 1) / tile * tile;
  *splits = (np + *chunk - 1) / *chunk;
}

}  // namespace yr

using namespace yr;

extern "C" size_t yr_hip_token_logprobs_workspace(int rows, int n_valid, int top_n, int dtype) {
  if (rows <= 0 || n_valid <= 0 || top_n < 0) return 0;
  int splits, chunk;
  logprobs_plan(rows, n_valid, dtype, &splits, &chunk);
  return splits > 1 ? kTicketBytes + (size_t)rows * splits * (3 + top_n) * sizeof(uint64_t) : 0;
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
  LogprobArgs a{x, tokens, logprob, entropy, top_logprob, top_ids, nullptr, nullptr, row_stride, n_valid, top_n, 1, 0};
  logprobs_plan(rows, n_valid, dtype, &a.splits, &a.chunk);
  const size_t need = yr_hip_token_logprobs_workspace(rows, n_valid, top_n, dtype);
  if (need > workspace_bytes || (need && !workspace))
    return fail(YR_E_WORKSPACE, "%s: workspace %zu < %zu", nm, workspace_bytes, need);
  if ((long long)rows * a.splits > 0x7fffffff) return fail(YR_E_INVALID, "%s: too many rows", nm);
  a.tickets = (uint32_t*)workspace;
  a.records = need ? (uint64_t*)((char*)workspace + kTicketBytes) : nullptr;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * a.splits));
  const size_t lds = (size_t)a.splits * top_n * sizeof(uint64_t);
  if (dtype == YR_DTYPE_F16)
    hipLaunchKernelGGL((logprobs_kernel<YR_DTYPE_F16>), grid, dim3(LP_THREADS), lds, st, a);
  else if (dtype == YR_DTYPE_BF16)
    hipLaunchKernelGGL((logprobs_kernel<YR_DTYPE_BF16>), grid, dim3(LP_THREADS), lds, st, a);
  else
    hipLaunchKernelGGL((logprobs_kernel<YR_DTYPE_F32>), grid, dim3(LP_THREADS), lds, st, a);
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
