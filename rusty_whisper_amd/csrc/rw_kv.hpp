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

#include <type_traits>

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

typedef float f4 __attribute__((ext_vector_type(4)));

// the pool's (and the logits') types: a conversion rounds to nearest even
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

// KV_ROWS rows x KV_COLS values of k and of v per workgroup, 8 values of a row
// per thread.  k's go straight to their rows; v's cross through LDS, so that
// neighbouring lanes have neighbouring rows, which are neighbours in a page
// where the rows are a prompt's.  Workgroups of one XCD (every eighth) take
// tiles that follow each other, whose parts of a cache line then meet in one L2.
// 24 prompts of 1500 rows, 1280 bf16 values: 112 us, the 4.9 TB/s of a large
// copy (tiles of 64 x 64 119, of 64 x 32 126, and 135 without the order); 64 rows
// of a step 5.0 us (tiles of 8 x 256 the same).
constexpr int KV_ROWS = 32, KV_COLS = 64;
template <class E>
__global__ __launch_bounds__(256) void k_kv_write(PagedView w, const float *__restrict__ k, int64_t ldk,
                                                  const float *__restrict__ v, int64_t ldv, int rows,
                                                  const int32_t *__restrict__ pos, int col_tiles, int tiles, int row0) {
  using T = typename E::T;
  typedef T Out __attribute__((ext_vector_type(8)));
  __shared__ T sv[KV_COLS][KV_ROWS + 2];
  __shared__ int64_t page0[KV_ROWS];  // where the row's page begins, -1: no place
  __shared__ int slot[KV_ROWS];
  const int tile = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);  // gridDim.x: a multiple of 8
  if (tile >= tiles) return;
  const int n = w.heads * w.dim, P = 1 << w.pr, t = threadIdx.x;
  const int r0 = row0 + tile / col_tiles * KV_ROWS, c0 = tile % col_tiles * KV_COLS;
  if (t < KV_ROWS) {
    int64_t at = -1;
    if (r0 + t < rows) {
      const int32_t *table = paged_row(w, r0 + t);
      const int p = pos[r0 + t];
      if (table && p >= 0 && (p >> w.pr) < w.ld) {
        const int page = table[p >> w.pr];
        if ((unsigned)page < (unsigned)w.n_pages) at = (int64_t)page * n << w.pr;
        slot[t] = p & (P - 1);
      }
    }
    page0[t] = at;
  }
  const int i = t / (KV_COLS / 8), c = c0 + t % (KV_COLS / 8) * 8;
  const bool in = r0 + i < rows && c < n;
  Out ok;
  if (in) {
    const float *a = k + (int64_t)(r0 + i) * ldk + c, *b = v + (int64_t)(r0 + i) * ldv + c;
    const f4 a0 = *(const f4 *)a, a1 = *(const f4 *)(a + 4), b0 = *(const f4 *)b, b1 = *(const f4 *)(b + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ok[j] = E::round(j < 4 ? a0[j] : a1[j - 4]);
      sv[c - c0 + j][i] = E::round(j < 4 ? b0[j] : b1[j - 4]);
    }
  }
  __syncthreads();
  if (in && page0[i] >= 0) {
    const int h = c / w.dim, d = c % w.dim;
    *(Out *)((T *)w.k + page0[i] + (((int64_t)h << w.pr) + slot[i]) * w.dim + d) = ok;
  }
#pragma unroll
  for (int j = 0; j < KV_ROWS * KV_COLS / 256; ++j) {
    const int e = j * 256 + t, row = e % KV_ROWS, col = e / KV_ROWS;
    if (c0 + col < n && page0[row] >= 0) ((T *)w.v)[page0[row] + ((int64_t)(c0 + col) << w.pr) + slot[row]] = sv[col][row];
  }
}

// Page copies whose ids travel in the launch's own arguments: no buffer that
// must outlive the call, and a captured launch keeps its ids.
constexpr int KV_PAIRS = 448;  // 3.5 KB of the 4 KB a launch's arguments may take
struct KvPairs {
  int2 id[KV_PAIRS];  // src, dst
};

// 16-byte pieces of page id[y], layer z / 2 of k (z even) or v; a page has
// `piece` of them per layer.  700 pages of 1.57 MB over 24 layers: 430 us, 5.1
// TB/s read and written, a large copy's rate.
__global__ __launch_bounds__(256) void k_kv_copy(uint4 *k, uint4 *v, int64_t piece, int64_t n_pages, KvPairs pairs) {
  uint4 *base = (blockIdx.z & 1 ? v : k) + (int64_t)(blockIdx.z >> 1) * n_pages * piece;
  const int2 id = pairs.id[blockIdx.y];
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < piece) base[id.y * piece + i] = base[id.x * piece + i];
}

// ------------------------------------------------------------- attention
//
// One workgroup of PA_WAVES wavefronts per (row, key/value head, 16 of its
// query heads, chunk of the row's keys).  A wavefront takes every PA_WAVES-th
// tile of keys (32 of a 2-byte type, 16 of f32: 1 KB of k and of v per 16
// values of the head) and keeps its own running maximum, sum and 16 x DH
// output; the wavefronts are joined through LDS at the end, chunks by
// k_paged_join.
//
// Lane 16h + r of a wavefront.  Scores come transposed, S = K q^T, so that a
// lane holds its query r's scores of keys 8h .. 8h + 7 (f32: 4h .. 4h + 3):
// just what the second product's left operand wants of lane (h, r), and v,
// whose rows are innermost, gives the right operand's 8 (4) keys of value
// 16 i + r as one 16-byte load.  So k and v go from memory to the matrix
// cores without LDS and without moves between lanes:
//   2-byte  v_mfma 16x16x32, A = 16 keys: row r of half s is key
//           8 (r / 4) + 4 s + r % 4, whose scores then lie in lane r / 4's
//           registers 4 s + r % 4.  The f32 q enters as 3 parts of the pool's
//           type, a product each; p as 3 bf16 for both types, as weights need
//           f32's range, and f16's v as 2 bf16 (8 and 3 bits).
//   f32     v_mfma 16x16x4 f32, A = 16 keys in order, exact products.
// Query columns beyond the group's are zeros (a matrix instruction costs the
// same with 1 or 16 queries, and the matrix cores are a quarter busy at most).
//
// Bound by reading k and v once: 131071 f16 keys of 8 heads of 128, 537 MB, 96 us
// (5.6 TB/s; counters: 555 MB, each line once) + 5 for the join.  61 rows of up
// to 8190 bf16 keys, 767 MB, 158 + 5 us: the rest is the tail of unlike rows.
// Measured and left (with two f16 parts of p and q): 8 wavefronts per workgroup
// (same: one CU draws about 50 GB/s either way), 3 wavefronts per SIMD (same; bf16
// spills), non-temporal loads (99 -> 113 us: half lines that the next
// wavefront's tile needs are gone), two or four neighbouring tiles per wavefront
// (98 -> 111).

constexpr int PA_WAVES = 4;
constexpr float PA_LOG2E = 1.44269504088896340736f;
// The running maximum m is only raised when a score passes it by PA_SLACK (in
// powers of two): then and only then the wavefront's lanes exchange their
// maxima and scale what they hold.  So p is at most 2^5, the maximum's at least
// 1, and a wavefront's sum l of them at least 1.
//   What a wavefront, a chunk hands on is its mean of v, sum p v / l, with m and
// l: means of finite values are finite, and weighted means of means too.  Only a
// wavefront's own sum p v can pass f32's range, of bf16 or f32 values near its
// end (WIDE): where a mean comes out infinite or NaN, the wavefront goes over its keys
// again with p at PA_LOW, and takes those means from there.  (Weights of 2^-30
// in the first place lost values below 2^-72, and p below 2^-96.)
constexpr float PA_SLACK = 5.0f;
constexpr float PA_LOW = 0x1p-40f;  // sums of 2^35 values stay in range

template <class E>
struct PaTile;  // keys per tile and lane, parts of an f32 operand, the two products

template <class E>
struct PaTile2 {
  using T = typename E::T;
  typedef T Op __attribute__((ext_vector_type(8)));
  static constexpr int KEYS = 32, PER = 8, STEP = 32, SUB = 2;  // STEP: values of the head per k operand
};
// f16's range is short: each further part of an operand is MOVE times what is left,
// and the parts' products have sums of their own (SUMS).  So q keeps 24 bits of
// every value down to 2^-37 of the query's largest, and something of it down to
// 2^-61.  (Two parts at one scale kept 22 bits down to 2^-18, nothing below 2^-40.)
template <>
struct PaTile<F16> : PaTile2<F16> {
  static constexpr int PARTS = 3, SUMS = 3;
  static constexpr float MOVE = 0x1p11f;
  static constexpr bool WIDE = false;
  static __device__ T part(float x) { return F16::round(x); }
  static __device__ f4 mma(Op a, Op b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct PaTile<BF16> : PaTile2<BF16> {
  static constexpr int PARTS = 3, SUMS = 1;
  static constexpr float MOVE = 1.0f;
  static constexpr bool WIDE = true;
  // x's 8 leading bits: three parts are all of f32's 24, and none is beyond the
  // type's largest (which a rounded one is for x above 3.39e38)
  static __device__ T part(float x) { return __builtin_bit_cast(T, (uint16_t)(__float_as_uint(x) >> 16)); }
  static __device__ f4 mma(Op a, Op b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct PaTile<F32> {
  using T = float;
  typedef f4 Op;
  static constexpr int KEYS = 16, PER = 4, STEP = 16, SUB = 1, PARTS = 1, SUMS = 1;
  static constexpr float MOVE = 1.0f;
  static constexpr bool WIDE = true;
  static __device__ T part(float x) { return x; }
  static __device__ f4 mma(Op a, Op b, f4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// x as a sum of PARTS operands, the p-th MOVE^p of its own size
template <class E>
__device__ inline void pa_parts(const float (&x)[PaTile<E>::PER], typename PaTile<E>::Op (&o)[PaTile<E>::PARTS]) {
#pragma unroll
  for (int j = 0; j < PaTile<E>::PER; ++j) {
    float rest = x[j];
#pragma unroll
    for (int p = 0; p < PaTile<E>::PARTS; ++p) {
      const typename E::T t = PaTile<E>::part(rest);
      o[p][j] = t;
      rest = (rest - (float)t) * PaTile<E>::MOVE;  // exact
    }
  }
}

// f16 values as sums of two bf16: the 8 leading bits and the 3 others
__device__ inline void pa_split(PaTile<F16>::Op x, PaTile<BF16>::Op &hi, PaTile<BF16>::Op &lo) {
  typedef uint32_t U4 __attribute__((ext_vector_type(4)));
  constexpr uint32_t HIGH = 0xFFFF0000u, HIGHS = 0x07060302u;  // v_perm: the upper halves of two registers
  U4 a, b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x0 = (float)x[2 * j], x1 = (float)x[2 * j + 1];
    const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
    a[j] = __builtin_amdgcn_perm(u1, u0, HIGHS);
    b[j] = __builtin_amdgcn_perm(__float_as_uint(x1 - __uint_as_float(u1 & HIGH)),
                                 __float_as_uint(x0 - __uint_as_float(u0 & HIGH)), HIGHS);
  }
  hi = __builtin_bit_cast(PaTile<BF16>::Op, a), lo = __builtin_bit_cast(PaTile<BF16>::Op, b);
}

// o += p v for a tile's weights and 16 ND values.  f16: all six products of the
// parts, so p v is as exact as in f32 at any size of p.  (In f16 parts, p at 2^10
// of the maximum, a weight below 2^-13 of the maximum lost bits and one below
// 2^-35 was nothing, though the sum had it: 162 us for 61 rows of up to 8190 keys,
// 8 heads of 128 with 4 query heads each, now 164; 16000 keys of 8 rows with 20
// query heads each, 126 and 136.  The f32 matrix instruction on converted v
// takes 170 and 145.)
template <class E, int ND>
__device__ inline void pa_add(const float (&p)[PaTile<E>::PER], const typename PaTile<E>::Op (&v)[ND], f4 (&o)[ND]) {
  using W = PaTile<std::conditional_t<sizeof(typename E::T) == 2, BF16, E>>;
  typename W::Op pf[W::PARTS];
  pa_parts<std::conditional_t<sizeof(typename E::T) == 2, BF16, E>>(p, pf);
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    if constexpr (std::is_same_v<E, F16>) {
      typename W::Op hi, lo;
      pa_split(v[i], hi, lo);
#pragma unroll
      for (int k = W::PARTS - 1; k >= 0; --k) o[i] = W::mma(pf[k], lo, o[i]), o[i] = W::mma(pf[k], hi, o[i]);
    } else {
#pragma unroll
      for (int k = 0; k < W::PARTS; ++k) o[i] = W::mma(pf[k], v[i], o[i]);
    }
  }
}

// a mean of finite values, rounded past f32's largest, is that
__device__ inline float pa_largest(float x) { return __builtin_copysignf(__FLT_MAX__, x); }

// exp2(x) for x <= 0 or -inf against a maximum that may be -inf itself
__device__ inline float pa_weight(float m, float top) {
  return m == -__builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

// ONE: a key head of one query head, which stands in all 16 columns, so that every
// lane has the weights of its keys and multiplies them with its v in f32, 8 fused
// multiply-adds per 16 values (o: of value 16 i + r, this lane's keys).  For f16,
// where the other form splits v: 448 keys of 5 rows, 20 heads of 64: 6.4 us against
// 7.8; 48 rows of up to 1500: 31.3 and 33; 300 rows of up to 700, 4 heads of 32: 11.6
// and 14.9; 61 rows of up to 8190, 8 heads of 128: 156 and 158.
template <class E, int DH, bool ONE>
__global__ __launch_bounds__(64 * PA_WAVES, 2) void k_paged_attn(
    const void *__restrict__ kp, const void *__restrict__ vp, const float *__restrict__ q, const int32_t *__restrict__ table,
    const int32_t *__restrict__ seq, const int32_t *__restrict__ lens, float *__restrict__ out, float *__restrict__ part,
    int rows, int kv_heads, int group, int pr, int n_pages, int n_seqs, int64_t ld_table, int64_t ldq, int64_t ldo,
    int max_len, int chunk) {
  using M = PaTile<E>;
  using Op = typename M::Op;
  using T = typename E::T;
  constexpr int NC = DH / M::STEP, ND = DH / 16, KEYS = M::KEYS, PER = M::PER, SUB = M::SUB, PARTS = M::PARTS;
  constexpr int LD = DH + 4;
  constexpr float NEG_INF = -__builtin_huge_valf();
  __shared__ float so[PA_WAVES][16][LD], sm[PA_WAVES][16], sl[PA_WAVES][16];

  // (row, key/value head) items; the query tiles of one item run eight
  // workgroups apart, on one XCD, whose L2 the second reads k and v from
  const int qtiles = (group + 15) / 16;
  const int qi = blockIdx.x / 8 % qtiles, item = blockIdx.x / (8 * qtiles) * 8 + blockIdx.x % 8;
  const int hk = item % kv_heads, row = item / kv_heads;
  if (row >= rows) return;
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int gq = min(16, group - 16 * qi);  // query heads of this tile
  const int heads = kv_heads * group, hq = hk * group + 16 * qi;
  const int sq = seq ? seq[row] : row;
  const int64_t most = ld_table << pr;
  int n = min(lens[row], max_len);
  if (n > most) n = (int)most;
  if ((unsigned)sq >= (unsigned)n_seqs) n = 0;
  float *orow = out + row * ldo + (int64_t)hq * DH;
  if (n <= 0) {
    if (blockIdx.y == 0)
      for (int i = threadIdx.x; i < gq * DH; i += 64 * PA_WAVES) orow[i] = 0.0f;
    return;
  }
  const int k0 = blockIdx.y * chunk;
  if (k0 >= n) return;
  const bool direct = n <= chunk;
  const int32_t *tab = table + (int64_t)sq * ld_table;
  const int end = (min(n, k0 + chunk) + KEYS - 1) / KEYS;
  const int P = 1 << pr;

  // where tile t's pages begin for this head (the two halves of a 32-key tile
  // lie in two 16-row pages), and which halves hold no rows
  struct Where {
    int64_t off0, off1;
    bool bad0, bad1;
  };
  auto where = [&](int t) __attribute__((always_inline)) {
    Where w;
    const int i = t * KEYS >> pr;
    int p0 = tab[i], p1 = p0;
    if (KEYS > 16 && pr == 4 && t * KEYS + 16 < n) p1 = tab[i + 1];
    w.bad0 = (unsigned)p0 >= (unsigned)n_pages, w.bad1 = (unsigned)p1 >= (unsigned)n_pages;
    w.off0 = (((int64_t)(w.bad0 ? 0 : p0) * kv_heads + hk) << pr) * DH;
    w.off1 = (((int64_t)(w.bad1 ? 0 : p1) * kv_heads + hk) << pr) * DH;
    return w;
  };
  const T *kb = (const T *)kp, *vb = (const T *)vp;
  Op kf[SUB][NC], vf[ND];
  auto load_k = [&](int t, const Where &w) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int kk = SUB == 1 ? r : 8 * (r >> 2) + 4 * s + (r & 3);
      const int slot = KEYS > 16 && pr == 4 ? kk & 15 : (t * KEYS & (P - 1)) + kk;
      const T *p = kb + (KEYS > 16 && kk >= 16 ? w.off1 : w.off0) + slot * DH + M::PER * h;
#pragma unroll
      for (int c = 0; c < NC; ++c) kf[s][c] = *(const Op *)(p + M::STEP * c);
    }
  };
  auto load_v = [&](int t, const Where &w) __attribute__((always_inline)) {
    const int kk = PER * h;
    const int slot = KEYS > 16 && pr == 4 ? kk & 15 : (t * KEYS & (P - 1)) + kk;
    const T *p = vb + (KEYS > 16 && kk >= 16 ? w.off1 : w.off0) + (r << pr) + slot;
#pragma unroll
    for (int i = 0; i < ND; ++i) vf[i] = *(const Op *)(p + ((16 * i) << pr));
  };

  const int t0 = k0 / KEYS + wv;
  int t = t0;
  Where now{};
  if (t < end) now = where(t), load_k(t, now);

  // q, in the scores' operand order; f16: each query's values scaled by a
  // power of two so that the largest lies in [2^14, 2^15), undone in `c`
  Op qf[PARTS][NC];
  float c = PA_LOG2E / __builtin_sqrtf((float)DH);
  {
    float x[NC][PER], top = 0.0f;
    const float *p = q + row * ldq + (int64_t)(hq + min(r, gq - 1)) * DH + PER * h;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < PER; j += 4) {
        const f4 y = *(const f4 *)(p + M::STEP * i + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][j + e] = ONE || r < gq ? y[e] : 0.0f, top = fmaxf(top, __builtin_fabsf(x[i][j + e]));
      }
    int e = 0;
    if (std::is_same_v<E, F16>) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      e = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
      c = ldexpf(c, e);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      Op o[PARTS];
      if (std::is_same_v<E, F16>)
#pragma unroll
        for (int j = 0; j < PER; ++j) x[i][j] = ldexpf(x[i][j], -e);
      pa_parts<E>(x[i], o);
#pragma unroll
      for (int k = 0; k < PARTS; ++k) qf[k][i] = o[k];
    }
  }

  for (float scale = 1.0f;; scale = PA_LOW) {
    std::conditional_t<ONE, float, f4> o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] = {};
    float m = NEG_INF, sum = 0.0f;  // query r's; sum: of this lane's keys

    for (; t < end; t += PA_WAVES) {
      load_v(t, now);
      const bool more = t + PA_WAVES < end;
      Where next{};
      if (more) next = where(t + PA_WAVES);
      f4 s[M::SUMS][SUB];
#pragma unroll
      for (int k = 0; k < M::SUMS; ++k)
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[k][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < PARTS; ++k)
#pragma unroll
          for (int u = 0; u < SUB; ++u) s[k % M::SUMS][u] = M::mma(kf[u][i], qf[k][i], s[k % M::SUMS][u]);
      if (more) load_k(t + PA_WAVES, next);
      float x[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        x[j] = s[M::SUMS - 1][j >> 2][j & 3];
#pragma unroll
        for (int k = M::SUMS - 2; k >= 0; --k) x[j] = fmaf(x[j], 1.0f / M::MOVE, s[k][j >> 2][j & 3]);
        x[j] *= c;
      }
      // keys behind the length, or in a page outside the pool, have no weight,
      // and what v holds there (anything) is taken as zero
      if ((t + 1) * KEYS > n || now.bad0 || now.bad1) {
        const bool bad = KEYS > 16 && h >= 2 ? now.bad1 : now.bad0;
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (bad || t * KEYS + PER * h + j >= n) {
            x[j] = NEG_INF;
#pragma unroll
            for (int i = 0; i < ND; ++i) vf[i][j] = (T)0.0f;
          }
      }
      float top = x[0];
#pragma unroll
      for (int j = 1; j < PER; ++j) top = fmaxf(top, x[j]);
      if (__builtin_amdgcn_ballot_w64(top > m + PA_SLACK)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float up = fmaxf(m, top), f = pa_weight(m, up);
        m = up;
        sum *= f;
        std::conditional_t<ONE, float, f4> fr;
        if constexpr (ONE) fr = f;
        else
#pragma unroll
          for (int i = 0; i < 4; ++i) fr[i] = __shfl(f, 4 * h + i);
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] *= fr;
      }
      const float base = m == NEG_INF ? 0.0f : m;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        x[j] = __builtin_amdgcn_exp2f(x[j] - base);
        if (M::WIDE) x[j] *= scale;
        sum += x[j];
      }
      if constexpr (ONE) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int j = 0; j < PER; ++j) o[i] = fmaf(x[j], (float)vf[i][j], o[i]);
      } else {
        pa_add<E>(x, vf, o);
      }
      now = next;
    }

    // the wavefront's means
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const bool first = scale == 1.0f;
    if (first && h == 0) sm[wv][r] = m, sl[wv][r] = sum;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // 0: no keys
    if constexpr (ONE) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        o[d] += __shfl_xor(o[d], 16);
        o[d] += __shfl_xor(o[d], 32);
        if (h == 0) so[wv][0][16 * d + r] = o[d] * inv;
      }
      break;
    } else {
      bool over = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int qr = 4 * h + i;
        const float f = __shfl(inv, qr);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const float y = o[d][i] * f;
          float &mean = so[wv][qr][16 * d + r];
          if (!M::WIDE || first) mean = y;
          else if (!__builtin_isfinite(mean)) mean = __builtin_isinf(y) && __builtin_isfinite(o[d][i]) ? pa_largest(y) : y;
          over |= qr < gq && !__builtin_isfinite(y);
        }
      }
      if (!M::WIDE || !first || !__builtin_amdgcn_ballot_w64(over)) break;
      t = t0;
      if (t < end) now = where(t), load_k(t, now);
    }
  }
  __syncthreads();

  // the wavefronts' means, each with its share of the weights
  const int64_t runs = (int64_t)rows * heads * gridDim.y;
  for (int i = threadIdx.x; i < gq * DH; i += 64 * PA_WAVES) {
    const int qr = i / DH, d = i % DH;
    float top = sm[0][qr], l = 0.0f, y = 0.0f, w[PA_WAVES];
#pragma unroll
    for (int k = 1; k < PA_WAVES; ++k) top = fmaxf(top, sm[k][qr]);
#pragma unroll
    for (int k = 0; k < PA_WAVES; ++k) l += w[k] = sl[k][qr] * pa_weight(sm[k][qr], top);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // 0: no page of the row is in the pool
#pragma unroll
    for (int k = 0; k < PA_WAVES; ++k) y += so[k][qr][d] * (w[k] * inv);
    if (M::WIDE && __builtin_isinf(y)) {
      bool finite = true;
#pragma unroll
      for (int k = 0; k < PA_WAVES; ++k) finite &= (bool)__builtin_isfinite(so[k][qr][d]);
      if (finite) y = pa_largest(y);
    }
    if (direct) {
      orow[i] = y;
    } else {
      const int64_t run = ((int64_t)row * heads + hq + qr) * gridDim.y + blockIdx.y;
      part[run * DH + d] = y;
      if (d == 0) part[runs * DH + 2 * run] = top, part[runs * DH + 2 * run + 1] = l;
    }
  }
}

// The chunks of one (row, query head): out = sum_z y_z w_z / sum_z w_z of their
// means y_z, w_z = l_z 2^(m_z - m).  A row of one chunk was written by
// k_paged_attn.  The chunks' weights go to LDS; then SIDE groups of threads, four values each, sum every
// SIDE-th chunk in order, and the groups' sums are added in order.
constexpr int PA_MAX_SPLIT = 512;  // chunks of a row at most: one row alone, two workgroups per CU
template <int DH>
__global__ __launch_bounds__(256) void k_paged_join(const float *__restrict__ part, const int32_t *__restrict__ seq,
                                                    const int32_t *__restrict__ lens, int n_seqs, int64_t most,
                                                    int max_len, int chunk, int nsplit, int heads, int64_t runs,
                                                    float *__restrict__ out, int64_t ldo) {
  constexpr int W = DH <= 32 ? 8 : DH <= 64 ? 16 : 32, SIDE = 256 / W;  // W threads of 4 values
  __shared__ float sw[PA_MAX_SPLIT], sl[4];
  __shared__ f4 sy[SIDE][DH / 4];
  const int row = blockIdx.x / heads, hq = blockIdx.x % heads;
  int n = min(lens[row], max_len);
  if (n > most) n = (int)most;
  if ((unsigned)(seq ? seq[row] : row) >= (unsigned)n_seqs || n <= chunk) return;
  const int nz = (n + chunk - 1) / chunk;  // <= nsplit <= PA_MAX_SPLIT
  const int64_t run0 = (int64_t)blockIdx.x * nsplit;
  const float *ml = part + runs * DH + 2 * run0;
  float top = -__builtin_huge_valf(), l = 0.0f;
  for (int z = threadIdx.x & 63; z < nz; z += 64) top = fmaxf(top, ml[2 * z]);
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
  for (int z = threadIdx.x; z < nz; z += 256) {
    const float w = ml[2 * z + 1] * pa_weight(ml[2 * z], top);
    sw[z] = w;
    l += w;
  }
  for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
  if ((threadIdx.x & 63) == 0) sl[threadIdx.x >> 6] = l;
  __syncthreads();
  l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int g = threadIdx.x / W, d = threadIdx.x % W;
  if (d < DH / 4) {
    f4 y{0.0f, 0.0f, 0.0f, 0.0f};
    const f4 *o = (const f4 *)(part + run0 * DH) + d;
#pragma unroll 4
    for (int z = g; z < nz; z += SIDE) y += o[z * (DH / 4)] * (sw[z] * inv);
    sy[g][d] = y;
  }
  __syncthreads();
  if (threadIdx.x < DH) {
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < SIDE; ++i) y += ((const float *)sy[i])[threadIdx.x];
    if (__builtin_isinf(y)) {
      bool finite = true;
      for (int z = 0; z < nz; ++z) finite &= (bool)__builtin_isfinite(part[(run0 + z) * DH + threadIdx.x]);
      if (finite) y = pa_largest(y);
    }
    out[row * ldo + (int64_t)hq * DH + threadIdx.x] = y;
  }
}

#endif  // __HIPCC__

}  // namespace rw
