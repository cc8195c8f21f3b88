// rw_score.hpp -- log-probs of given tokens, entropy and top alternatives of
// rows of logits.
//
// With M = max x, S = sum e^(x - M), T = sum (x - M) e^(x - M):
//   lp(t) = x_t - M - ln S,   entropy = ln S - T / S
// (both terms of the entropy are non-negative, so nothing cancels).
#pragma once
#include "rw_kv.hpp"

namespace rw {

constexpr int SCORE_TOP = 32;  // alternatives per row at most

#if defined(__HIPCC__)

__device__ inline float score_max(float v, float *scratch) {
  for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
}
__device__ inline float score_sum(float v, float *scratch) {
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}
__device__ inline int score_imin(int v, int *scratch) {
  for (int o = 1; o < 64; o <<= 1) v = min(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return min(min(scratch[0], scratch[1]), min(scratch[2], scratch[3]));
}

// One workgroup per row, which reads the row for the maximum, for the sums
// and once per alternative.
template <class E>
__global__ __launch_bounds__(256) void k_score_row(const typename E::T *__restrict__ logits, int64_t ld, int n,
                                                   const uint32_t *__restrict__ tokens, int64_t n_tok,
                                                   float *__restrict__ logprobs, float *__restrict__ entropy, int k,
                                                   uint32_t *__restrict__ top_ids, float *__restrict__ top_lp) {
  constexpr float NEG_INF = -__builtin_huge_valf();
  __shared__ float sf[4];
  __shared__ int si[4];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  const typename E::T *x = logits + row * ld;
  float m = NEG_INF;
  for (int i = t; i < n; i += 256) m = fmaxf(m, E::load(x + i));
  m = score_max(m, sf);
  float s = 0.0f, u = 0.0f;
  for (int i = t; i < n; i += 256) {
    const float d = E::load(x + i) - m, e = expf(d);
    s += e;
    if (e != 0.0f) u += d * e;  // also NaN
  }
  s = score_sum(s, sf);
  u = score_sum(u, sf);
  const float ls = logf(s);
  const bool bad = !(s > 0.0f);  // NaN: a NaN or +inf among the logits, or only -inf
  if (t == 0 && entropy) entropy[row] = bad ? __builtin_nanf("") : ls - u / s;
  for (int64_t i = t; i < n_tok; i += 256) {
    const uint32_t id = tokens[row * n_tok + i];
    float lp = __builtin_nanf("");
    if (id == 0xFFFFFFFFu) lp = 0.0f;
    else if (id < (uint32_t)n && !bad) lp = (E::load(x + id) - m) - ls;
    logprobs[row * n_tok + i] = lp;
  }
  float pv = __builtin_huge_valf();
  int pi = -1;
  for (int j = 0; j < k; ++j) {
    float bv = NEG_INF;
    int bi = INT32_MAX;
    for (int i = t; i < n && !bad; i += 256) {
      const float v = E::load(x + i);
      if ((v < pv || (v == pv && i > pi)) && v > bv) bv = v, bi = i;
    }
    const float mv = score_max(bv, sf);
    const int mi = score_imin(bv == mv ? bi : INT32_MAX, si);
    if (t == 0) {
      top_ids[row * k + j] = mi == INT32_MAX ? 0xFFFFFFFFu : (uint32_t)mi;
      top_lp[row * k + j] = bad ? __builtin_nanf("") : mi == INT32_MAX ? NEG_INF : (mv - m) - ls;
    }
    pv = mv, pi = mi;
  }
}

#endif  // __HIPCC__

}  // namespace rw
