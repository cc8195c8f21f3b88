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
// One workgroup per row, three passes over it, the second and third out of the
// caches: M; a histogram of weights (and counts, for top-k) over the logits, linear
// from M down to where weights end; and the tokens of the few bins in which the questions fall (where
// does the count reach k, the weight top_p of all, the weight u of the kept),
// which are then ordered among themselves.  Bins of many tokens get
// histograms of their own, those of equal logits histograms over ids.
#pragma once
#include "rw_kv.hpp"
#include "rw_rocm.h"
#include "rw_serve.hpp"

namespace rw {

constexpr size_t SAMPLE_VOCAB = (size_t)1 << 20;
constexpr int SAMPLE_THREADS = 512;
constexpr int SAMPLE_BITS = 42;  // of a weight
constexpr int SAMPLE_BINS = 4096, SAMPLE_SUB = 1024;
constexpr int SAMPLE_LIST = 512;   // tokens ordered at once: a thread each
constexpr uint32_t SAMPLE_NONE = 0xFFFFFFFFu;

struct SampleArgs {
  const float *u, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  uint32_t *tokens;
  float *logprobs;
  int64_t ld;
  int n, rows;
};

#if defined(__HIPCC__)

// 2^y, -64 <= y <= 0: y = k + r, and a polynomial for 2^r, |r| <= 1/2, whose largest
// relative error is the least of its degree (1.1e-12, 2^-39.7).  The coefficients are held
// in scalar registers: the compiler moves each into a vector register before its
// product, three instructions for one.
struct SampleSeries {
  double c[8];
  __device__ SampleSeries() {
    constexpr double k[] = {1.3175858116190163e-06, 1.5309737422254016e-05, 0.00015403851748721433, 0.001333345206224751,
                            0.009618128542862396,   0.05550410939341712,    0.2402265069888037,     0.6931471805465141};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = k[i];
      asm volatile("" : "+s"(c[i]));
    }
  }
  __device__ double exp2(double y) const {
    // y rounded to whole numbers by adding what leaves no bits for more; k's own bits
    // then go to the exponent (conversions, roundings and ldexp of 64 bits run at a quarter of the rate)
    const double n = y + 0x1.8p52, r = y - (n - 0x1.8p52);
    double p = __builtin_fma(r, c[0], c[1]);
#pragma unroll
    for (int i = 2; i < 8; ++i) p = __builtin_fma(p, r, c[i]);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + (__builtin_bit_cast(uint64_t, n) << 52));
  }
};

// How a row's logits weigh, and which bin of the first histogram they are in.
struct SampleScale {
  float top, cut;  // M, and the smallest logit that is kept
  double step;     // log2 e / t
  float bins;      // per half a logit
  SampleSeries e;

  // (of a logit from `cut` on; of others, anything)
  __device__ uint64_t weight(float x) const {
    const double w = e.exp2(((double)x - (double)top) * step);
    // 2^10 + w has the bits of w down to 2^-42
    return __builtin_bit_cast(uint64_t, w + 1024.0) - __builtin_bit_cast(uint64_t, 1024.0);
  }
  // half the distance to M (no two logits are too far apart for that), in bins
  __device__ float place(float x) const { return __builtin_fmaf(x, -0.5f, 0.5f * top) * bins; }
  __device__ int bin(float x) const { return (int)fminf(place(x), (float)(SAMPLE_BINS - 1)); }
};

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

struct SampleFound {  // a bin, its tokens and their weight, and what precedes it
  unsigned long long before_w, w;
  unsigned int before_c, c;
  int bin;
};

struct alignas(16) SampleToken {
  float x;
  int id;
  unsigned long long w;
};

struct SampleShared {
  SampleHist<SAMPLE_BINS> all;
  SampleHist<SAMPLE_SUB> sub;
  unsigned long long ww[SAMPLE_THREADS / 64];
  unsigned int wc[SAMPLE_THREADS / 64];
  float fx[SAMPLE_THREADS / 64], fy[SAMPLE_THREADS / 64];
  SampleFound found;
  SampleToken list[SAMPLE_LIST];  // to be ordered
  unsigned int n_list;
  SampleAt at;
};

// A row: its whole 16-byte vectors, read in batches of B per thread, all of a batch
// on their way at once and without branches between them (loads under branches wait
// for each other); and the few logits before and behind those.
template <class E>
struct SampleRow {
  using T = typename E::T;
  static constexpr int V = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(V)));
  const T *x;
  int n, first, vecs;  // logits; those before the first vector; vectors

  __device__ SampleRow(const T *row, int n_vocab) : x(row), n(n_vocab) {
    first = min(n, (int)((16 - ((uintptr_t)x & 15)) % 16 / sizeof(T)));
    vecs = (n - first) / V;
  }
  // f(V logits, the first one's id) for every vector of this thread, and some of
  // -inf; those before and behind the vectors come singly, with -inf beside them
  template <int B, class F>
  __device__ __forceinline__ void each(F f) const {
    constexpr T NONE = (T)-__builtin_huge_valf();
    const Vec *body = (const Vec *)(x + first);
#pragma unroll 1
    for (int g0 = 0; g0 < vecs; g0 += B * SAMPLE_THREADS) {
      const int g = g0 + (int)threadIdx.x;
      Vec v[B];
#pragma unroll
      for (int b = 0; b < B; ++b) v[b] = body[min(g + b * SAMPLE_THREADS, vecs - 1)];
      if (g0 + B * SAMPLE_THREADS > vecs) {
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int i = 0; i < V; ++i) v[b][i] = g + b * SAMPLE_THREADS < vecs ? v[b][i] : NONE;
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        float y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = (float)v[b][i];
        f(y, first + (g + b * SAMPLE_THREADS) * V);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int e = (int)threadIdx.x < first ? (int)threadIdx.x : vecs * V + (int)threadIdx.x;
    if ((int)(threadIdx.x & ~63u) < first + V) {  // (whole wavefronts)
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = (float)NONE;
      if (e < n) y[0] = (float)x[e];
      f(y, e);
    }
  }
  // the same one by one
  template <int B, class F>
  __device__ __forceinline__ void each_one(F f) const {
    each<B>([&](const float(&y)[V], int id) {
#pragma unroll
      for (int i = 0; i < V; ++i) f(y[i], id + i);
    });
  }
};

// the workgroup's largest value, in every thread
__device__ inline float sample_max(float v, float *s) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) v = fmaxf(v, __shfl_xor(v, x));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[threadIdx.x & (SAMPLE_THREADS / 64 - 1)];
#pragma unroll
  for (int x = 1; x < SAMPLE_THREADS / 64; x <<= 1) v = fmaxf(v, __shfl_xor(v, x));
  __syncthreads();
  return v;
}

// What the bins of this thread weigh, what precedes them, and all of it
template <int BINS>
struct SampleSums {
  static constexpr int PER = BINS / SAMPLE_THREADS;
  const SampleHist<BINS> &h;
  uint64_t own_w, w, total_w;
  uint32_t own_c, c, total_c;

  __device__ SampleSums(const SampleHist<BINS> &hist, SampleShared &s) : h(hist) {
    constexpr int WAVES = SAMPLE_THREADS / 64;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    own_w = 0, own_c = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = threadIdx.x * PER + (k + threadIdx.x) % PER;  // (lanes' bins in as many banks)
      own_w += h.w[i], own_c += h.c[i];
    }
    w = own_w, c = own_c;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const uint64_t a = __shfl_up((unsigned long long)w, x);
      const uint32_t b = __shfl_up(c, x);
      if (lane >= x) w += a, c += b;
    }
    if (lane == 63) s.ww[wv] = w, s.wc[wv] = c;
    __syncthreads();
    w -= own_w, c -= own_c, total_w = 0, total_c = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      if (i < wv) w += s.ww[i], c += s.wc[i];
      total_w += s.ww[i], total_c += s.wc[i];
    }
    __syncthreads();
  }
  // the bin in which the weight (or the count) reaches `want` (> 0, <= the total)
  __device__ void find(bool by_count, uint64_t want, SampleFound &f) const {
    if (by_count ? c < want && c + own_c >= want : w < want && w + own_w >= want) {
      uint64_t aw = w, bw = 0;
      uint32_t ac = c, bc = 0;
      int i = threadIdx.x * PER - 1;
      do ++i, aw += bw, ac += bc, bw = h.w[i], bc = h.c[i];
      while (by_count ? ac + bc < want : aw + bw < want);
      f = SampleFound{aw, bw, ac, bc, i};
    }
  }
};

// The tokens of lo .. hi that f names into the list, as many as it takes; how many there are
template <int B, class E, class F>
__device__ __forceinline__ int sample_gather(const SampleRow<E> &row, const SampleScale &c, SampleShared &s, float lo, float hi, F f) {
  constexpr int V = SampleRow<E>::V;
  if (threadIdx.x == 0) s.n_list = 0;
  __syncthreads();
  row.template each<B>([&](const float(&y)[V], int id) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < V; ++i) any |= (y[i] >= lo) & (y[i] <= hi);
    if (any)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (y[i] >= lo && y[i] <= hi && f(y[i], id + i)) {
          const unsigned at = atomicAdd(&s.n_list, 1u);
          if (at < SAMPLE_LIST) s.list[at].x = y[i], s.list[at].id = id + i;
        }
  });
  __syncthreads();
  const int m = (int)s.n_list;
  if ((int)threadIdx.x < min(m, SAMPLE_LIST)) s.list[threadIdx.x].w = c.weight(s.list[threadIdx.x].x);
  __syncthreads();
  return m;
}

// The place at which the weight (the count) reaches `want`, among the listed tokens,
// which follow what `b` says precedes them
__device__ __forceinline__ SampleAt sample_place(SampleShared &s, int m, const SampleFound &b, bool by_count, uint64_t want) {
  if ((int)threadIdx.x < m) {
    const SampleToken own = s.list[threadIdx.x];
    uint64_t w = b.before_w;
    uint32_t n = b.before_c;
#pragma unroll 8
    for (int e = 0; e < m; ++e) {
      const SampleToken y = s.list[e];
      const bool in = (y.x > own.x) | ((y.x == own.x) & (y.id < own.id));
      w += in ? y.w : 0, n += in;
    }
    if (by_count ? n + 1 == want : w < want && w + own.w >= want) s.at = SampleAt{w + own.w, own.x, own.id};
  }
  __syncthreads();
  const SampleAt at = s.at;
  __syncthreads();
  return at;
}

// The same in a bin of too many tokens, which are narrowed by histograms: over the
// bin's logits, and where they are equal over the ids
template <class E>
__device__ __forceinline__ SampleAt sample_narrow(const SampleRow<E> &row, const SampleScale &c, SampleShared &s, SampleFound b,
                                                  bool by_count, uint64_t want) {
  const int first = b.bin;
  float hi = -__builtin_huge_valf(), lo = hi;  // the bin's own logits; lo: the largest -x
  row.template each_one<1>([&](float x, int) {
    if (x >= c.cut && c.bin(x) == first) hi = fmaxf(hi, x), lo = fmaxf(lo, -x);
  });
  hi = sample_max(hi, s.fx), lo = -sample_max(lo, s.fy);
  int i0 = 0, i1 = row.n;
  do {
    const bool ids = !(lo < hi);
    // (hi is in the first bin, lo in the last, whatever they are, in 64 bits: every turn takes one of them away)
    const double f = ids ? 0.0 : (double)SAMPLE_SUB / ((double)hi - (double)lo);
    const int shift = max(0, 32 - __builtin_clz((unsigned)(i1 - i0 - 1) | 1) - 10);
    auto sub_bin = [&](float x, int id) {
      return ids ? (id - i0) >> shift : min(SAMPLE_SUB - 1, (int)(((double)hi - (double)x) * f));
    };
    for (int i = threadIdx.x; i < SAMPLE_SUB; i += SAMPLE_THREADS) s.sub.w[i] = 0, s.sub.c[i] = 0;
    __syncthreads();
    row.template each_one<1>([&](float x, int id) {
      if (x >= lo && x <= hi && id >= i0 && id < i1) {
        const int k = sub_bin(x, id);
        atomicAdd(&s.sub.w[k], (unsigned long long)c.weight(x));
        atomicAdd(&s.sub.c[k], 1u);
      }
    });
    __syncthreads();
    const SampleSums<SAMPLE_SUB> o(s.sub, s);
    o.find(by_count, want - (by_count ? b.before_c : b.before_w), s.found);
    __syncthreads();
    const SampleFound g = s.found;
    __syncthreads();
    b.before_w += g.before_w, b.before_c += g.before_c, b.c = g.c;
    if (ids) {
      i1 = min(i1, i0 + ((g.bin + 1) << shift)), i0 += g.bin << shift;
    } else {
      float h2 = -__builtin_huge_valf(), l2 = h2;
      row.template each_one<1>([&](float x, int id) {
        if (x >= lo && x <= hi && sub_bin(x, id) == g.bin) h2 = fmaxf(h2, x), l2 = fmaxf(l2, -x);
      });
      hi = sample_max(h2, s.fx), lo = -sample_max(l2, s.fy);
    }
  } while (b.c > SAMPLE_LIST);
  const int m = sample_gather<1>(row, c, s, lo, hi, [&](float, int id) { return id >= i0 && id < i1; });
  return sample_place(s, m, b, by_count, want);
}

__device__ inline uint64_t sample_share(float p, uint64_t w) {  // the least sum that has p of w
  return max((uint64_t)1, min(w, (uint64_t)__builtin_ceil((double)fmaxf(p, 0.0f) * (double)w)));
}
__device__ inline uint64_t sample_past(float u, uint64_t w) {  // the least sum above u of w
  return min(w, (uint64_t)__builtin_floor((double)fminf(fmaxf(u, 0.0f), 1.0f) * (double)w) + 1);
}

struct SampleAsk {
  int top_k;
  float top_p, u;
};
struct SampleAnswer {
  SampleAt at;
  uint64_t kept;
  bool done;
};
// The three questions in turn: the weight of the first top_k, of these the weight that top_p
// keeps, and the token at u of that; f(bin, by_count, want, &place) answers one, or not
template <class F>
__device__ __forceinline__ SampleAnswer sample_answer(SampleShared &s, const SampleSums<SAMPLE_BINS> &all, const SampleAsk &a, F f) {
  SampleAnswer g{SampleAt{all.total_w, 0.0f, 0}, 0, true};
#pragma unroll 1
  for (int q = 0; q < 3 && g.done; ++q) {
    if (q == 0 ? a.top_k <= 0 || (uint32_t)a.top_k >= all.total_c : q == 1 && !(a.top_p < 1.0f)) continue;
    if (q == 2) g.kept = g.at.sum;
    const uint64_t want = q == 0 ? (uint64_t)a.top_k : q == 1 ? sample_share(a.top_p, g.at.sum) : sample_past(a.u, g.at.sum);
    all.find(q == 0, want, s.found);
    __syncthreads();
    const SampleFound b = s.found;
    g.done = f(b, q == 0, want, g.at);
  }
  return g;
}

// The same of m listed tokens that are all: each one's rank and sum, then the questions
__device__ __forceinline__ SampleAnswer sample_few(SampleShared &s, int m, const SampleAsk &a) {
  SampleToken own{};
  uint64_t w = 0, total = 0;
  uint32_t n = 0;
  const bool in = (int)threadIdx.x < m;
  if (in) {
    own = s.list[threadIdx.x];
#pragma unroll 8
    for (int e = 0; e < m; ++e) {
      const SampleToken y = s.list[e];
      const bool first = (y.x > own.x) | ((y.x == own.x) & (y.id < own.id));
      w += first ? y.w : 0, n += first, total += y.w;
    }
    if (threadIdx.x == 0) s.ww[0] = total;
  }
  __syncthreads();
  SampleAnswer g{SampleAt{s.ww[0], 0.0f, 0}, 0, true};
#pragma unroll 1
  for (int q = 0; q < 3; ++q) {
    if (q == 0 ? a.top_k <= 0 || a.top_k >= m : q == 1 && !(a.top_p < 1.0f)) continue;
    if (q == 2) g.kept = g.at.sum;
    const uint64_t want = q == 0 ? (uint64_t)a.top_k : q == 1 ? sample_share(a.top_p, g.at.sum) : sample_past(a.u, g.at.sum);
    if (in && (q == 0 ? n + 1 == want : w < want && w + own.w >= want)) s.at = SampleAt{w + own.w, own.x, own.id};
    __syncthreads();
    g.at = s.at;
    __syncthreads();
  }
  return g;
}

// ... where their bins have too many tokens.  A call: inlined, the kernel keeps 23 (f32), 30 (f16) or 32 (bf16)
// of a lane's registers in memory, so 8, 28 and 30, and 768 rows by top-p take 109 us, not 114
template <class E>
__device__ __noinline__ SampleAnswer sample_slow(const typename E::T *x, int n, float top, float cut, double step, float bins,
                                                 SampleShared &s, SampleAsk a) {
  const SampleRow<E> row(x, n);
  const SampleScale c{top, cut, step, bins, SampleSeries()};
  const SampleSums<SAMPLE_BINS> all(s.all, s);
  return sample_answer(s, all, a, [&](const SampleFound &b, bool by_count, uint64_t want, SampleAt &at) {
    at = sample_narrow(row, c, s, b, by_count, want);
    return true;
  });
}

template <class E>
__global__ __launch_bounds__(SAMPLE_THREADS, 4) void k_sample(const typename E::T *__restrict__ logits, SampleArgs a) {
  constexpr float INF = __builtin_huge_valf();
  constexpr int V = SampleRow<E>::V;
  __shared__ SampleShared s;
  const int64_t r = blockIdx.y * (int64_t)gridDim.x + blockIdx.x;
  if (r >= a.rows) return;
  const SampleRow<E> row(logits + r * a.ld, a.n);
  const float t = a.temperature ? a.temperature[r] : 1.0f, u = a.u[r];
  const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  for (int i = threadIdx.x; i < SAMPLE_BINS; i += SAMPLE_THREADS) s.all.w[i] = 0, s.all.c[i] = 0;
  for (int i = threadIdx.x; i < SAMPLE_SUB; i += SAMPLE_THREADS) s.sub.w[i] = 0, s.sub.c[i] = 0;
  float own = -INF;  // this thread's largest logit, or NaN
  row.template each<52 / V>([&](const float(&y)[V], int) {
#pragma unroll
    for (int i = 0; i < V; ++i) own = __builtin_elementwise_maximum(own, y[i]);
  });
  const float top = sample_max(own == own ? own : INF, s.fx);
  if (!(top > -INF && top < INF) || !(t < INF) || u != u || top_p != top_p || min_p != min_p) {
    if (threadIdx.x == 0) {
      a.tokens[r] = SAMPLE_NONE;
      if (a.logprobs) a.logprobs[r] = __builtin_nanf("");
    }
    return;
  }
  // the first of the order: also where no weight has min_p, those of the largest logits (1) neither
  if (t <= 0.0f || top_k == 1 || min_p > 1.0f) {
    int id = INT32_MAX;
    if (own == top)  // (few threads)
      row.template each_one<1>([&](float x, int i) {
        if (x == top) id = min(id, i);
      });
    const float least = -sample_max(own == top ? -(float)id : -INF, s.fy);  // (ids below 2^20 are exact)
    if (threadIdx.x == 0) {
      a.tokens[r] = (uint32_t)least;
      if (a.logprobs) a.logprobs[r] = 0.0f;
    }
    return;
  }
  // weights end 43 ln 2 below the top; those below min_p of it are not kept
  const double low = (double)top - 29.9 * (double)t;
  const double least = min_p > 0.0f ? fmax(low, (double)top + (double)t * log((double)min_p)) : low;
  float cut = (float)fmax(least, -(double)__FLT_MAX__);
  if ((double)cut < least) cut = -__int_as_float(__float_as_int(-cut) - (cut < 0.0f ? 1 : -1));  // the next above
  cut = fminf(cut, top);
  bool few = least > low;
  if (top_k > 0 && top_k <= SAMPLE_THREADS) {
    // the threads' largest logits: the top_k-th of these bounds the row's from below
    const float f = top > cut ? fminf((float)SAMPLE_SUB / (0.5f * top - 0.5f * cut), __FLT_MAX__) : 0.0f;
    const int k = own >= cut ? (int)fminf((0.5f * top - 0.5f * own) * f, (float)(SAMPLE_SUB - 1)) : -1;
    if (k >= 0) atomicAdd(&s.sub.c[k], 1u);
    __syncthreads();
    const SampleSums<SAMPLE_SUB> o(s.sub, s);
    if (o.total_c >= (uint32_t)top_k) {
      o.find(true, (uint64_t)top_k, s.found);
      __syncthreads();
      cut = -sample_max(k >= 0 && k <= s.found.bin ? -own : -INF, s.fy);
      few = true;
    }
  }
  const SampleScale c{top, cut, 1.4426950408889634074 / (double)t,
                      top > cut ? fminf((float)SAMPLE_BINS / (0.5f * top - 0.5f * cut), __FLT_MAX__) : 0.0f, SampleSeries()};
  const SampleAsk ask{top_k, top_p, u};
  SampleAnswer g;
  g.done = false;
  if (few) {  // what is left is ordered at once
    const int m = sample_gather<52 / V>(row, c, s, cut, top, [](float, int) { return true; });
    if (m <= SAMPLE_LIST) g = sample_few(s, m, ask);
  }
  if (!g.done) {
    const bool counts = top_k > 0;
    row.template each<16 / V>([&](const float(&y)[V], int) {
      bool any = false;
#pragma unroll
      for (int i = 0; i < V; ++i) any |= y[i] >= cut;
      if (any)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (y[i] >= cut) {
            const int b = c.bin(y[i]);
            atomicAdd(&s.all.w[b], (unsigned long long)c.weight(y[i]));
            if (counts) atomicAdd(&s.all.c[b], 1u);
          }
    });
    __syncthreads();
    const SampleSums<SAMPLE_BINS> all(s.all, s);
    g = sample_answer(s, all, ask, [&](const SampleFound &b, bool by_count, uint64_t want, SampleAt &at) {
      // the bin's logits lie in lo .. hi, by the error of its place in f32
      const double wide = 2.0 / (double)c.bins, end = (double)(b.bin + 1) * wide;
      const double err = 0x1p-21 * (__builtin_fabs((double)top) + end);
      const float hi = b.bin == 0 ? top : (float)((double)top - (double)b.bin * wide + err);
      const float lo = b.bin == SAMPLE_BINS - 1 || c.bins == 0.0f ? cut : fmaxf(cut, (float)((double)top - end - err));
      const int m = sample_gather<52 / V>(row, c, s, lo, hi, [&](float x, int) { return c.bin(x) == b.bin; });
      if (m <= SAMPLE_LIST) at = sample_place(s, m, b, by_count, want);
      return m <= SAMPLE_LIST;
    });
  if (!g.done) g = sample_slow<E>(row.x, row.n, top, cut, c.step, c.bins, s, ask);
  }
  if (threadIdx.x == 0) {
    a.tokens[r] = (uint32_t)g.at.id;
    if (a.logprobs)
      a.logprobs[r] = (float)(((double)g.at.x - (double)top) / (double)t - log(__builtin_ldexp((double)g.kept, -SAMPLE_BITS)));
  }
}

template <class E>
int sample_launch_of(const void *logits, const SampleArgs &a, size_t rows, hipStream_t s) {
  const size_t x = std::min(rows, (size_t)1 << 20);  // (2^32 threads side by side are too many for a launch)
  const dim3 grid((unsigned)x, (unsigned)cdiv(rows, x));
  hipLaunchKernelGGL((k_sample<E>), grid, dim3(SAMPLE_THREADS), 0, s, (const typename E::T *)logits, a);
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
