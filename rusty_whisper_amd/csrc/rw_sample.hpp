// rw_sample.hpp -- a token per row of logits: temperature, top-k, min-p, top-p, and
// the draw from a given uniform number.
//
// The order: larger logits first, equal ones by lowest id.  With M = max x and the
// temperature t, a token's weight is w = e^((x - M) / t).  Kept are the first k,
// those with w >= min_p, and of these the shortest beginning that has top_p of
// their weight; the token is the first whose weights' sum passes u times the kept ones'.
//
// Sums decide between tokens, so weights are formed in 64 bits and held as whole
// multiples of 2^-42: then no order of additions changes a sum (histograms by
// atomics give the same result every time), and 2^20 of them fit in 64 bits.
// A token below 2^-43 of the largest weighs nothing and is never drawn.
//
// One workgroup per row.  The row is read once and stays in registers (rows too
// long for that are read again).  A histogram of weights and counts over the
// logits, linear from M down to where weights end, is summed up once; each question
// (where does the count reach k, the weight top_p of all, the weight u of the kept) then
// names one bin, whose few tokens are ordered among themselves.  A bin of many
// tokens gets a histogram of its own, one of equal logits a histogram over ids.
#pragma once
#include "rw_kv.hpp"
#include "rw_rocm.h"
#include "rw_serve.hpp"

namespace rw {

constexpr size_t SAMPLE_VOCAB = (size_t)1 << 20;
constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_BITS = 42;  // of a weight
constexpr int SAMPLE_BINS = 4096, SAMPLE_SUB = 2048;
constexpr int SAMPLE_LIST = 512, SAMPLE_FEW = 128;  // tokens ordered at once: room for, and wanted
constexpr uint32_t SAMPLE_NONE = 0xFFFFFFFFu;

struct SampleArgs {
  const float *u, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  uint32_t *tokens;
  float *logprobs;
  int64_t ld;
  int n;
};

#if defined(__HIPCC__)

// e^y, y <= 0: y = k ln 2 + r, and 12 terms of the series of e^r, |r| <= 0.35
// (the rest is below 2^-47)
__device__ inline double sample_exp(double y) {
  y = fmax(y, -80.0);
  const double k = __builtin_rint(y * 1.4426950408889634074);
  double r = __builtin_fma(k, -0.693147180559945286227, y);
  r = __builtin_fma(k, -2.31904681384629956e-17, r);
  double p = 1.0 / 39916800.0;
  constexpr double c[] = {1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0,
                          1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,          1.0};
#pragma unroll
  for (int i = 0; i < 11; ++i) p = __builtin_fma(p, r, c[i]);
  return __builtin_ldexp(p, (int)k);
}

struct SampleAt {  // a place in the order
  uint64_t sum;    // weight up to it, its own included
  float x;
  int id;
};

template <int BINS>
struct SampleHist {
  unsigned long long w[BINS];
  unsigned int c[BINS];
};

struct SampleShared {
  SampleHist<SAMPLE_BINS> all;
  SampleHist<SAMPLE_SUB> sub;
  unsigned long long ww[SAMPLE_THREADS / 64];
  unsigned int wc[SAMPLE_THREADS / 64];
  float fx[SAMPLE_THREADS / 64], fy[SAMPLE_THREADS / 64];
  // what a question found: a bin, and what precedes it
  unsigned long long before_w;
  unsigned int before_c, count;
  int bin;
  // the tokens of a bin
  float lx[SAMPLE_LIST];
  int li[SAMPLE_LIST];
  unsigned long long lw[SAMPLE_LIST];
  unsigned int n_list;
  SampleAt at;
};

// E: the logits' type; NJ: 16-byte vectors per thread (0: the row is read again
// by every pass)
template <class E, int NJ>
struct SampleRow {
  using T = typename E::T;
  static constexpr int V = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(V)));
  const T *x;
  int n, skip, steps;
  Vec held[NJ ? NJ : 1];

  __device__ Vec load(int j) const {
    const int e0 = (j * SAMPLE_THREADS + (int)threadIdx.x) * V - skip;
    if (e0 >= 0 && e0 + V <= n) return *(const Vec *)(x + e0);
    Vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = e0 + i >= 0 && e0 + i < n ? x[e0 + i] : (T)-__builtin_huge_valf();
    return v;
  }
  __device__ void begin(const T *row, int n_vocab) {
    x = row, n = n_vocab;
    skip = (int)(((uintptr_t)x & 15) / sizeof(T));  // places count from the 16 bytes in which the row starts
    steps = (n + skip + SAMPLE_THREADS * V - 1) / (SAMPLE_THREADS * V);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (j < steps) held[j] = load(j);
  }
  // f(logit, id) for every token of this thread (places outside the row: -inf)
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (j < steps) {
#pragma unroll
          for (int i = 0; i < V; ++i) f((float)held[j][i], (j * SAMPLE_THREADS + (int)threadIdx.x) * V - skip + i);
        }
    } else {
      for (int j = 0; j < steps; ++j) {
        const Vec v = load(j);
#pragma unroll
        for (int i = 0; i < V; ++i) f((float)v[i], (j * SAMPLE_THREADS + (int)threadIdx.x) * V - skip + i);
      }
    }
  }
};

// the workgroup's largest value, in every thread
__device__ inline float sample_max(float v, float *s) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) v = fmaxf(v, __shfl_xor(v, x));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[threadIdx.x & (SAMPLE_THREADS / 64 - 1)];
#pragma unroll
  for (int x = 1; x < SAMPLE_THREADS / 64; x <<= 1) v = fmaxf(v, __shfl_xor(v, x));
  return v;
}

// What precedes this thread's BINS / 1024 bins (in their order), and all of it
struct SampleSums {
  uint64_t w, total_w;
  uint32_t c, total_c;
};
template <int BINS>
__device__ inline SampleSums sample_sums(const SampleHist<BINS> &h, SampleShared &s) {
  constexpr int PER = BINS / SAMPLE_THREADS, WAVES = SAMPLE_THREADS / 64;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  uint64_t w = 0;
  uint32_t c = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) w += h.w[threadIdx.x * PER + i], c += h.c[threadIdx.x * PER + i];
  const uint64_t own_w = w;
  const uint32_t own_c = c;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const uint64_t a = __shfl_up((unsigned long long)w, x);
    const uint32_t b = __shfl_up(c, x);
    if (lane >= x) w += a, c += b;
  }
  if (lane == 63) s.ww[wv] = w, s.wc[wv] = c;
  __syncthreads();
  SampleSums o{w - own_w, 0, c - own_c, 0};
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i < wv) o.w += s.ww[i], o.c += s.wc[i];
    o.total_w += s.ww[i], o.total_c += s.wc[i];
  }
  __syncthreads();
  return o;
}

// the bin in which the weight (or the count) reaches `want` (> 0, <= the total)
template <int BINS>
__device__ inline void sample_find(const SampleHist<BINS> &h, const SampleSums &o, bool by_count, uint64_t want, SampleShared &s) {
  constexpr int PER = BINS / SAMPLE_THREADS;
  uint64_t w = o.w;
  uint32_t c = o.c;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint64_t bw = h.w[threadIdx.x * PER + i];
    const uint32_t bc = h.c[threadIdx.x * PER + i];
    if (by_count ? c < want && c + bc >= want : w < want && w + bw >= want)
      s.bin = threadIdx.x * PER + i, s.before_w = w, s.before_c = c, s.count = bc;
    w += bw, c += bc;
  }
  __syncthreads();
}

template <class E, int NJ>
struct Sampler {
  SampleShared &s;
  const SampleRow<E, NJ> &row;
  float top, cut;  // M, and the smallest logit that is kept
  double t;
  float scale;     // bins per logit of the first histogram

  __device__ uint64_t weight(float x) const {
    const double w = sample_exp(((double)x - (double)top) / t);
    return (uint64_t)__builtin_rint(__builtin_ldexp(w, SAMPLE_BITS));
  }
  __device__ int bin(float x) const { return min(SAMPLE_BINS - 1, (int)((top - x) * scale)); }

  // The first place in the order where the weight (the count) reaches `want`
  __device__ SampleAt find(const SampleSums &all, bool by_count, uint64_t want) {
    sample_find(s.all, all, by_count, want, s);
    int b = s.bin;
    uint64_t before_w = s.before_w;
    uint32_t before_c = s.before_c, count = s.count;
    __syncthreads();
    // the bin's own logits
    float hi = -__builtin_huge_valf(), lo = hi;  // lo: the largest -x
    row.each([&](float x, int) {
      if (x >= cut && bin(x) == b) hi = fmaxf(hi, x), lo = fmaxf(lo, -x);
    });
    hi = sample_max(hi, s.fx), lo = -sample_max(lo, s.fy);
    int i0 = 0, i1 = row.n;
    while (count > SAMPLE_FEW && (lo < hi || count > SAMPLE_LIST)) {
      const bool ids = !(lo < hi);
      // (hi is in the first bin, lo in the last, whatever they are, in 64 bits: every turn takes one of them away)
      const double f = ids ? 0.0 : (double)SAMPLE_SUB / ((double)hi - (double)lo);
      const int shift = max(0, 32 - __builtin_clz((unsigned)(i1 - i0 - 1) | 1) - 11);
      auto sub_bin = [&](float x, int id) {
        return ids ? (id - i0) >> shift : min(SAMPLE_SUB - 1, (int)(((double)hi - (double)x) * f));
      };
      for (int i = threadIdx.x; i < SAMPLE_SUB; i += SAMPLE_THREADS) s.sub.w[i] = 0, s.sub.c[i] = 0;
      __syncthreads();
      row.each([&](float x, int id) {
        if (x >= lo && x <= hi && id >= i0 && id < i1) {
          const int k = sub_bin(x, id);
          atomicAdd(&s.sub.w[k], (unsigned long long)weight(x));
          atomicAdd(&s.sub.c[k], 1u);
        }
      });
      __syncthreads();
      const SampleSums o = sample_sums(s.sub, s);
      sample_find(s.sub, o, by_count, want - (by_count ? before_c : before_w), s);
      b = s.bin, before_w += s.before_w, before_c += s.before_c, count = s.count;
      __syncthreads();
      if (ids) {
        i1 = min(i1, i0 + ((b + 1) << shift)), i0 += b << shift;
      } else {
        float h2 = -__builtin_huge_valf(), l2 = h2;
        row.each([&](float x, int id) {
          if (x >= lo && x <= hi && sub_bin(x, id) == b) h2 = fmaxf(h2, x), l2 = fmaxf(l2, -x);
        });
        hi = sample_max(h2, s.fx), lo = -sample_max(l2, s.fy);
      }
    }
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    row.each([&](float x, int id) {
      if (x >= lo && x <= hi && id >= i0 && id < i1) {
        const unsigned at = atomicAdd(&s.n_list, 1u);
        if (at < SAMPLE_LIST) s.lx[at] = x, s.li[at] = id, s.lw[at] = weight(x);
      }
    });
    __syncthreads();
    const int m = min((int)s.n_list, SAMPLE_LIST);
    if ((int)threadIdx.x < m) {
      const float x = s.lx[threadIdx.x];
      const int id = s.li[threadIdx.x];
      const uint64_t own = s.lw[threadIdx.x];
      uint64_t w = before_w;
      uint32_t c = before_c;
      for (int e = 0; e < m; ++e)
        if (s.lx[e] > x || (s.lx[e] == x && s.li[e] < id)) w += s.lw[e], ++c;
      if (by_count ? c + 1 == want : w < want && w + own >= want) s.at = SampleAt{w + own, x, id};
    }
    __syncthreads();
    const SampleAt at = s.at;
    __syncthreads();
    return at;
  }
};

template <class E, int NJ>
__global__ __launch_bounds__(SAMPLE_THREADS) void k_sample(const typename E::T *__restrict__ logits, SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t r = blockIdx.x;
  SampleRow<E, NJ> row;
  row.begin(logits + r * a.ld, a.n);
  const float t = a.temperature ? a.temperature[r] : 1.0f, u = a.u[r];
  const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  constexpr float INF = __builtin_huge_valf();
  float top = -INF;
  bool nan = false;
  row.each([&](float x, int) {
    top = fmaxf(top, x);
    nan |= x != x;
  });
  top = sample_max(nan ? INF : top, s.fx);
  if (!(top > -INF && top < INF) || !(t < INF) || u != u || top_p != top_p || min_p != min_p) {
    if (threadIdx.x == 0) {
      a.tokens[r] = SAMPLE_NONE;
      if (a.logprobs) a.logprobs[r] = __builtin_nanf("");
    }
    return;
  }
  if (t <= 0.0f || top_k == 1) {  // the first of the order
    float id = -INF;
    row.each([&](float x, int i) {
      if (x == top) id = fmaxf(id, -(float)i);  // (ids below 2^20 are exact)
    });
    id = -sample_max(id, s.fy);
    if (threadIdx.x == 0) {
      a.tokens[r] = (uint32_t)id;
      if (a.logprobs) a.logprobs[r] = 0.0f;
    }
    return;
  }
  Sampler<E, NJ> m{s, row, top, -INF, (double)t, 0.0f};
  // weights end 43 ln 2 below the top; those below min_p of it are not kept
  const double low = (double)top - 29.9 * (double)t;
  const double least = min_p > 0.0f ? fmax(low, (double)top + (double)t * log((double)min_p)) : low;
  float cut = (float)fmax(least, -(double)__FLT_MAX__);
  if ((double)cut < least) cut = -__int_as_float(__float_as_int(-cut) - (cut < 0.0f ? 1 : -1));  // the next above
  m.cut = cut = fminf(cut, top);
  m.scale = top > cut ? (float)SAMPLE_BINS / (top - cut) : 0.0f;
  if (!(m.scale < INF)) m.scale = __FLT_MAX__;
  for (int i = threadIdx.x; i < SAMPLE_BINS; i += SAMPLE_THREADS) s.all.w[i] = 0, s.all.c[i] = 0;
  __syncthreads();
  row.each([&](float x, int) {
    if (x >= cut) {
      const uint64_t w = m.weight(x);
      const int b = m.bin(x);
      atomicAdd(&s.all.w[b], (unsigned long long)w);
      atomicAdd(&s.all.c[b], 1u);
    }
  });
  __syncthreads();
  const SampleSums all = sample_sums(s.all, s);
  uint64_t kept = all.total_w;
  if (top_k > 0 && (uint32_t)top_k < all.total_c) kept = m.find(all, true, (uint64_t)top_k).sum;
  if (top_p < 1.0f) {
    const double want = __builtin_ceil((double)fmaxf(top_p, 0.0f) * (double)kept);
    kept = m.find(all, false, max((uint64_t)1, min(kept, (uint64_t)want))).sum;
  }
  const double want = __builtin_floor((double)fminf(fmaxf(u, 0.0f), 1.0f) * (double)kept);
  const SampleAt at = m.find(all, false, min(kept, (uint64_t)want + 1));
  if (threadIdx.x == 0) {
    a.tokens[r] = (uint32_t)at.id;
    if (a.logprobs)
      a.logprobs[r] = (float)(((double)at.x - (double)top) / (double)t - log(__builtin_ldexp((double)kept, -SAMPLE_BITS)));
  }
}

template <class E>
int sample_launch_of(const void *logits, const SampleArgs &a, size_t rows, hipStream_t s) {
  const auto *x = (const typename E::T *)logits;
  constexpr int V = 16 / sizeof(typename E::T);
  const size_t steps = cdiv((size_t)a.n + V - 1, SAMPLE_THREADS * V);
#define RW_SAMPLE(NJ) hipLaunchKernelGGL((k_sample<E, NJ>), dim3((unsigned)rows), dim3(SAMPLE_THREADS), 0, s, x, a)
  if (steps <= 2) RW_SAMPLE(2);
  else if (steps <= 7) RW_SAMPLE(7);
  else if (steps <= 13) RW_SAMPLE(13);
  else RW_SAMPLE(0);
#undef RW_SAMPLE
  return launched("k_sample");
}

inline int sample_launch(int dtype, const void *logits, const SampleArgs &a, size_t rows, hipStream_t s) {
  switch (dtype) {
    case RW_F32: return sample_launch_of<F32>(logits, a, rows, s);
    case RW_F16: return sample_launch_of<F16>(logits, a, rows, s);
    default: return sample_launch_of<BF16>(logits, a, rows, s);
  }
}

#endif  // __HIPCC__

}  // namespace rw
