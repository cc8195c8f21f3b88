// rw_kv.hpp -- the paged key/value cache's kernels: rows into pages, copies of
// pages, attention of one token per row over its sequence's pages.
//
//   k  [layer][page][head][row][value]     v  [layer][page][head][value][row]
//
// (rw_rocm.h, rw_kv_pages).  Within a page and head, k's rows and v's values
// are contiguous runs.
#pragma once
#include <stddef.h>
#include <stdint.h>

#if defined(__HIPCC__)
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#endif

namespace rw {

// A layer's pages, and who holds them, as the kernels see them.
struct PagedView {
  const void *k, *v;     // the layer's pages
  int heads, dim, pr;    // key/value heads, values per head, log2(rows per page)
  int n_pages;
  const int32_t *table;  // [n_seqs][ld]
  int n_seqs;
  int64_t ld;
  const int32_t *seq;    // [rows], or null: row r is sequence r
};

#if defined(__HIPCC__)

struct F32 {
  using T = float;
  static __device__ float load(const T *p) { return *p; }
  static __device__ T round(float x) { return x; }
};
struct F16 {
  using T = _Float16;
  static __device__ float load(const T *p) { return (float)*p; }
  static __device__ T round(float x) { return (T)x; }
};
struct BF16 {
  using T = __bf16;
  static __device__ float load(const T *p) { return (float)*p; }
  static __device__ T round(float x) { return (T)x; }
};

// the table row of a call's row, or null where the table has none
__device__ inline const int32_t *paged_row(const PagedView &w, int r) {
  const int s = w.seq ? w.seq[r] : r;
  return (unsigned)s < (unsigned)w.n_seqs ? w.table + (int64_t)s * w.ld : nullptr;
}

// One value of one row per thread: k and v rounded to the pool's type.
template <class E>
__global__ __launch_bounds__(256) void k_kv_write(PagedView w, const float *__restrict__ k, int64_t ldk,
                                                  const float *__restrict__ v, int64_t ldv, int rows,
                                                  const int32_t *__restrict__ pos) {
  const int r = blockIdx.x, n = w.heads * w.dim, P = 1 << w.pr;
  const int32_t *table = paged_row(w, r);
  const int p = pos[r];
  if (!table || p < 0 || (p >> w.pr) >= w.ld) return;
  const int page = table[p >> w.pr], slot = p & (P - 1);
  if ((unsigned)page >= (unsigned)w.n_pages) return;
  const int64_t base = (int64_t)page * n << w.pr;
  auto *pk = (typename E::T *)w.k + base, *pv = (typename E::T *)w.v + base;
  for (int c = threadIdx.x; c < n; c += 256) {
    const int h = c / w.dim, d = c % w.dim;
    pk[(((int64_t)h << w.pr) + slot) * w.dim + d] = E::round(k[r * ldk + c]);
    pv[((int64_t)c << w.pr) + slot] = E::round(v[r * ldv + c]);
  }
}

// Page copies whose ids travel in the launch's own arguments: no buffer that
// must outlive the call, and a captured launch keeps its ids.
constexpr int KV_PAIRS = 448;  // 3.5 KB of the 4 KB a launch's arguments may take
struct KvPairs {
  int2 id[KV_PAIRS];  // src, dst
};

// 16-byte pieces of page id[y], layer z / 2 of k (z even) or v; a page has
// `piece` of them per layer.
__global__ __launch_bounds__(256) void k_kv_copy(uint4 *k, uint4 *v, int64_t piece, int64_t n_pages, KvPairs pairs) {
  uint4 *base = (blockIdx.z & 1 ? v : k) + (int64_t)(blockIdx.z >> 1) * n_pages * piece;
  const int2 id = pairs.id[blockIdx.y];
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < piece) base[id.y * piece + i] = base[id.x * piece + i];
}

// One wavefront per (row, query head): the softmax's running maximum and sum
// over 64 keys at a time, a lane per key for the scores, a lane per value for
// the products.
template <class E>
__global__ __launch_bounds__(64) void k_paged_attn(PagedView w, const float *__restrict__ q, int64_t ldq, int heads,
                                                   const int32_t *__restrict__ lens, int max_len, float scale,
                                                   float *__restrict__ out, int64_t ldo) {
  constexpr float NEG_INF = -__builtin_huge_valf();
  __shared__ float sq[128], sp[64];
  const int r = blockIdx.x / heads, h = blockIdx.x % heads, hk = h / (heads / w.heads), l = threadIdx.x, P = 1 << w.pr;
  const int32_t *table = paged_row(w, r);
  const int64_t most = w.ld << w.pr;
  int n = min(lens[r], max_len);
  if (n > most) n = (int)most;
  float *o = out + r * ldo + (int64_t)h * w.dim;
  if (!table || n <= 0) {
    for (int d = l; d < w.dim; d += 64) o[d] = 0.0f;
    return;
  }
  for (int d = l; d < w.dim; d += 64) sq[d] = q[r * ldq + (int64_t)h * w.dim + d] * scale;
  __syncthreads();
  const auto *pk = (const typename E::T *)w.k, *pv = (const typename E::T *)w.v;
  float m = NEG_INF, sum = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int t0 = 0; t0 < n; t0 += 64) {
    const int t = t0 + l;
    float s = NEG_INF;
    if (t < n) {
      const int page = table[t >> w.pr];
      if ((unsigned)page < (unsigned)w.n_pages) {
        const auto *row = pk + ((((int64_t)page * w.heads + hk) << w.pr) + (t & (P - 1))) * w.dim;
        s = 0.0f;
        for (int d = 0; d < w.dim; ++d) s = fmaf(sq[d], E::load(row + d), s);
      }
    }
    float mx = s;
    for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
    const float mn = fmaxf(m, mx);
    if (mn == NEG_INF) continue;
    const float f = expf(m - mn), p = expf(s - mn);
    float ps = p;
    for (int x = 1; x < 64; x <<= 1) ps += __shfl_xor(ps, x);
    sum = sum * f + ps;
    m = mn;
    __syncthreads();
    sp[l] = p;
    __syncthreads();
    const int top = min(64, n - t0);
    for (int i = 0; i < 2; ++i) {
      const int d = l + 64 * i;
      if (d >= w.dim) break;
      float a = acc[i] * f;
      for (int j = 0; j < top; ++j) {
        if (sp[j] == 0.0f) continue;  // also a page outside the pool
        const int page = table[(t0 + j) >> w.pr];
        a = fmaf(sp[j], E::load(pv + ((((int64_t)page * w.heads + hk) * w.dim + d) << w.pr) + ((t0 + j) & (P - 1))), a);
      }
      acc[i] = a;
    }
  }
  for (int i = 0; i < 2; ++i)
    if (l + 64 * i < w.dim) o[l + 64 * i] = sum > 0.0f ? acc[i] / sum : 0.0f;
}

#endif  // __HIPCC__

}  // namespace rw
