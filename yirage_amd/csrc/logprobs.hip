// Log probabilities of given tokens, the distribution's entropy and its top
// alternatives, of rows of logits x (f16, bf16 or fp32):
//
//   m = max x, s = sum e^(x - m), logprob = x[token] - m - log s,
//   H = -sum p log p = log s - sum e^(x - m) (x - m) / s,
//   the `top` largest values, equal ones by the lowest index.
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
  long long stride;  // elements between rows
  int n, top;
};

constexpr int LP_THREADS = 1024;
constexpr int LP_MAX_TOP = 64;

template <int DT>
__device__ __forceinline__ float logit(const void* x, long long i) {
  if constexpr (DT == YR_DTYPE_F32) return gptr((const float*)x)[i];
  else return ld_elem<DT>(gptr((const uint16_t*)x)[i]);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// (value, index) order of the alternatives: larger value, then lower index.
__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

template <int DT>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(LogprobArgs a) {
  constexpr int W = LP_THREADS / kWave, kNone = 0x7fffffff;
  __shared__ float s_v[W];
  __shared__ int s_i[W];
  __shared__ double s_s[W], s_t[W];
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid / kWave;
  const char* x = (const char*)a.x + (size_t)row * a.stride * (DT == YR_DTYPE_F32 ? 4 : 2);
  // the `top` best in order, one pass each; the first one is the maximum
  float lv = INFINITY, m = -INFINITY;
  int li = -1;
  for (int k = 0; k < max(a.top, 1); k++) {
    float bv = -INFINITY;
    int bi = kNone;
    for (int i = tid; i < a.n; i += LP_THREADS) {
      const float v = logit<DT>(x, i);
      if ((k == 0 || better(lv, li, v, i)) && v == v && (bi == kNone || better(v, i, bv, bi))) {
        bv = v;
        bi = i;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float ov = __shfl_xor(bv, o, kWave);
      const int oi = __shfl_xor(bi, o, kWave);
      if (oi != kNone && (bi == kNone || better(ov, oi, bv, bi))) {
        bv = ov;
        bi = oi;
      }
    }
    if (tid % kWave == 0) {
      s_v[wave] = bv;
      s_i[wave] = bi;
    }
    __syncthreads();
    bv = s_v[0];
    bi = s_i[0];
    for (int w = 1; w < W; w++)
      if (s_i[w] != kNone && (bi == kNone || better(s_v[w], s_i[w], bv, bi))) {
        bv = s_v[w];
        bi = s_i[w];
      }
    __syncthreads();
    if (k == 0) m = bv;
    if (k < a.top && tid == 0) {
      a.top_lp[(size_t)row * a.top + k] = bi == kNone ? -INFINITY : bv;
      a.top_ids[(size_t)row * a.top + k] = bi == kNone ? -1 : bi;
    }
    lv = bi == kNone ? -INFINITY : bv;
    li = bi;
  }
  double s = 0, t = 0;
  for (int i = tid; i < a.n; i += LP_THREADS) {
    const float y = logit<DT>(x, i) - m, e = __expf(y);
    s += e;
    t += e == 0.f ? 0.f : e * y;
  }
  s = wave_sum_d(s);
  t = wave_sum_d(t);
  if (tid % kWave == 0) {
    s_s[wave] = s;
    s_t[wave] = t;
  }
  __syncthreads();
  s = t = 0;
  for (int w = 0; w < W; w++) {
    s += s_s[w];
    t += s_t[w];
  }
  const double ls = log(s);
  if (tid == 0) {
    const int64_t tok = a.tokens[row];
    a.logprob[row] = tok < 0 || tok >= a.n ? NAN : (float)((double)(logit<DT>(x, tok) - m) - ls);
    a.entropy[row] = (float)(ls - t / s);
  }
  for (int k = tid; k < a.top; k += LP_THREADS) {
    const size_t at = (size_t)row * a.top + k;
    if (a.top_ids[at] >= 0) a.top_lp[at] = (float)((double)(a.top_lp[at] - m) - ls);
  }
}

}  // namespace yr

using namespace yr;

extern "C" int yr_hip_token_logprobs(const void* x, const int64_t* tokens, float* logprob, float* entropy,
                                     float* top_logprob, int64_t* top_ids, int rows, int n, int n_valid,
                                     int64_t row_stride, int top_n, int dtype, void* stream) {
  const char* nm = "yr_hip_token_logprobs";
  if (!x || !tokens || !logprob || !entropy || (top_n > 0 && (!top_logprob || !top_ids)))
    return fail(YR_E_INVALID, "%s: null pointer", nm);
  if (rows <= 0 || n <= 0 || n_valid <= 0 || n_valid > n || row_stride < n) return fail(YR_E_INVALID, "%s: bad shape", nm);
  if (top_n < 0 || top_n > LP_MAX_TOP || top_n > n_valid)
    return fail(YR_E_INVALID, "%s: top_n %d (at most %d and the valid columns)", nm, top_n, LP_MAX_TOP);
  LogprobArgs a{x, tokens, logprob, entropy, top_logprob, top_ids, row_stride, n_valid, top_n};
  hipStream_t st = (hipStream_t)stream;
#define YR_LP(DT_)        \
  if (dtype == DT_)       \
    hipLaunchKernelGGL((logprobs_kernel<DT_>), dim3(rows), dim3(LP_THREADS), 0, st, a);
  YR_LP(YR_DTYPE_F16) else YR_LP(YR_DTYPE_BF16) else YR_LP(YR_DTYPE_F32) else return fail(YR_E_INVALID, "%s: dtype", nm);
#undef YR_LP
  YR_CHECK_LAUNCH(nm);
  return YR_OK;
}
