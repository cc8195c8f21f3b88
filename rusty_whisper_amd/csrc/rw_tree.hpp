// rw_tree.hpp -- attention of several new tokens per sequence over keys and values
// in pages: trees of drafted tokens (a mask), chunks of prompts (each token sees
// those before it), and single tokens over 8-bit pages.
//
// Row j of tree i sees the rows 0 .. past - 1 of its sequence and, of the tree's own
// (rows past .. past + nodes - 1 of the sequence), those that its mask's bits name, or 0 .. j
// without a mask.  The queries of a tree and key head (rows x query heads of the
// head) are counted together and cut into tiles of 16: the columns of the scores'
// products, as in rw_kv.hpp, whose operands, precision and treatment of sums this
// follows; 8-bit pools differ:
//   keys    as f16, which has all their values, times q in 2 f16 parts (22 bits and
//           more of every value down to 2^-29 of its query's largest); the score times the key's
//           scale and, where q is small, what brings q back to its own size
//   values  as bf16, which has them too, times p s (p: the weight, s: the value's
//           scale) in 3 bf16 parts, all of its bits down to 2^-109; so s enters at 2^40 times its
//           size, and may be any number that f32 has.  (In 2, 5e-6 of the results was off; in 2 f16
//           parts, of the largest p s at 2^10 .. 2^15, as little as in 3, but a small weight
//           lost bits where the value of a large one is zero, and int8 has many zeros.)
// f16 pools: q in those 2 parts, not 3; of p's 3 parts against v's 2 the product of the
// least two, 2^-24 of the whole, is left out.
#pragma once
#include "rw_kv8.hpp"

namespace rw {

#if defined(__HIPCC__)

// 8 values of a pool of 8 bits, as f16 and as bf16: both exact
template <class E>
struct Kv8;
template <>
struct Kv8<I8> {
  static __device__ PaTile<F16>::Op f16(u32x2 a) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // x + 128 below the bits of 1024: 1152 + x
      const uint32_t u = a[i >> 1] ^ 0x80808080u;
      const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, i & 1 ? 0x04030402u : 0x04010400u);
      const h2 x = __builtin_bit_cast(h2, b) - (_Float16)1152.0f;
      o[i] = __builtin_bit_cast(uint32_t, x);
    }
    return __builtin_bit_cast(PaTile<F16>::Op, o);
  }
  static __device__ PaTile<BF16>::Op bf16(u32x2 a) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = a[i >> 1] ^ 0x80808080u;  // x + 128: bytes without a sign have their own conversions
      const float x0 = (float)(i & 1 ? u >> 16 & 0xFF : u & 0xFF) - 128.0f, x1 = (float)(i & 1 ? u >> 24 : u >> 8 & 0xFF) - 128.0f;
      o[i] = __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), 0x07060302u);
    }
    return __builtin_bit_cast(PaTile<BF16>::Op, o);
  }
  static constexpr bool FINITE = true;  // no code is an infinity or a NaN
};
template <>
struct Kv8<E4M3> {
  static __device__ PaTile<F16>::Op f16(u32x2 a) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = i & 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a[i >> 1], 1.0f, true))
                   : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a[i >> 1], 1.0f, false));
    return __builtin_bit_cast(PaTile<F16>::Op, o);
  }
  static __device__ PaTile<BF16>::Op bf16(u32x2 a) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = i & 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a[i >> 1], 1.0f, true))
                   : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a[i >> 1], 1.0f, false));
    return __builtin_bit_cast(PaTile<BF16>::Op, o);
  }
  static constexpr bool FINITE = false;
};

// the first c bytes of a word (none, some or all)
__device__ inline uint32_t kv8_first(int c) { return c <= 0 ? 0 : c >= 4 ? ~0u : (1u << (8 * c)) - 1; }
// which bytes of a word are e4m3's NaN, which become zeros
__device__ inline uint32_t kv8_take_nan(uint32_t &w) {
  const uint32_t x = ((w & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u;
  w &= ~(x * 0xFFu);
  return (x | x >> 7 | x >> 14 | x >> 21) & 0xFu;
}

struct TreeArgs {
  const void *k, *v;
  const float *ks, *vs;
  const float *q;
  float *out, *part;
  const int32_t *table, *seq, *starts, *past;
  const uint32_t *mask;
  int64_t ldq, ldo, ld_table;
  int n_words, rows, n_trees, max_rows, kv_heads, group, pr, n_pages, n_seqs, max_len, chunk, qtiles;
};

// What tree i of a call is: its first row, its rows in this launch, the rows of
// the sequence before it, the rows it may see, its row of the table.  (An end below
// zero is taken as zero: its distance from the first row could pass 32 bits and come out positive.)
struct TreeSpan {
  int start, rows, past, n;
  const int32_t *table;
};
__device__ inline TreeSpan tree_span(const TreeArgs &a, int i) {
  constexpr int MOST = 1 << 30;
  TreeSpan s;
  const int sq = a.seq ? a.seq[i] : i;
  const int most = (int)min((int64_t)min(MOST, a.max_len), a.ld_table << a.pr);
  s.past = min(a.past[i], MOST);
  int nodes = 0;
  if (a.starts) {
    s.start = a.starts[i];
    nodes = s.start < 0 ? 0 : max(0, min(max(a.starts[i + 1], 0), a.rows) - s.start);
    s.rows = min(nodes, a.max_rows);
  } else {
    s.start = i, s.rows = 1;
  }
  s.n = s.past < 0 || (unsigned)sq >= (unsigned)a.n_seqs ? 0 : min(s.past + nodes, most);
  s.table = a.table + (int64_t)((unsigned)sq < (unsigned)a.n_seqs ? sq : 0) * a.ld_table;
  return s;
}
// the end of the keys that the queries u0 .. u1 - 1 of a tree see
__device__ inline int tree_end(const TreeArgs &a, const TreeSpan &s, int u1) {
  if (!a.starts || a.mask) return s.n;
  return min(s.n, s.past + (u1 - 1) / a.group + 1);
}
// Bits 0 .. PER - 1: whether a row (`node` of its tree, `mask` its words) sees the
// keys a0 .. a0 + PER - 1
template <int PER>
__device__ inline uint32_t tree_sees(const TreeArgs &a, const TreeSpan &s, const uint32_t *mask, int node, int a0) {
  constexpr uint32_t ALL = PER == 32 ? ~0u : (1u << PER) - 1;
  const int b = a0 - s.past;
  uint32_t bits = ALL;
  if (b > -PER && a.starts) {
    if (!a.mask) {
      const int c = node + 1 - b;  // how many of them
      bits = c <= 0 ? 0 : c >= PER ? ALL : (1u << c) - 1;
    } else {
      const int w = max(b, 0) >> 5;
      const uint32_t lo = w < a.n_words ? mask[w] : 0, hi = w + 1 < a.n_words ? mask[w + 1] : 0;
      const uint64_t both = ((uint64_t)hi << 32) | lo;
      bits = b < 0 ? (lo << -b) | ((1u << -b) - 1) : (uint32_t)(both >> (b & 31));
    }
  }
  const int c = s.n - a0;
  return bits & (c <= 0 ? 0 : c >= PER ? ALL : (1u << c) - 1);
}

// c + how many of a lane's 8 keys both bits are set of
__device__ inline f4 tree_count(uint32_t w, uint32_t v, f4 c) {
  PaTile<BF16>::Op a, b;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a[j] = (__bf16)(w >> j & 1 ? 1.0f : 0.0f);
    b[j] = (__bf16)(v >> j & 1 ? 1.0f : 0.0f);
  }
  return PaTile<BF16>::mma(a, b, c);
}
// x as two f16, the second at 2^11 of its own size
__device__ inline void tree_q_halves(const float (&x)[8], PaTile<F16>::Op &hi, PaTile<F16>::Op &lo) {
#pragma unroll
  for (int j = 0; j < 8; ++j) hi[j] = (_Float16)x[j], lo[j] = (_Float16)((x[j] - (float)hi[j]) * 0x1p11f);
}
// weights as 3 bf16
__device__ inline void tree_parts(const float *p, PaTile<BF16>::Op (&pf)[3]) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = p[j];
  pa_parts<BF16>(x, pf);
}
// o += p v, p in 3 bf16 parts, v as 2
__device__ inline f4 tree_split_mma(const PaTile<BF16>::Op (&p)[3], PaTile<BF16>::Op hi, PaTile<BF16>::Op lo, f4 o) {
  o = PaTile<BF16>::mma(p[2], hi, o);
  o = PaTile<BF16>::mma(p[1], lo, o);
  o = PaTile<BF16>::mma(p[1], hi, o);
  o = PaTile<BF16>::mma(p[0], lo, o);
  return PaTile<BF16>::mma(p[0], hi, o);
}

// How a pool's tiles of keys enter the two products.  Lane 16 h + r of a
// wavefront holds of a tile's KEYS keys the scores of PER h .. PER h + PER - 1 for
// query r, and their values 16 i + r.
template <class E, int DH>
struct TreeTile {
  using M = PaTile<E>;
  using T = typename E::T;
  using QOp = typename M::Op;   // of the scores' product
  static constexpr bool SCALED = false, WIDE = M::WIDE;
  static constexpr int KEYS = M::KEYS, SUB = M::SUB, PER = 4 * SUB, STEPS = DH / M::STEP;
  static constexpr bool HALF = std::is_same_v<E, F16>;
  static constexpr int PARTS = HALF ? 2 : M::PARTS, SUMS = HALF ? 2 : M::SUMS;
  static constexpr int VAL = M::PER;  // values per lane and step
  static constexpr float MOVE = M::MOVE;
  static constexpr int HEAD = DH;
  typename M::Op kr[SUB][STEPS], vr[DH / 16];
  // the first value of step c for the lanes of `h`
  static __device__ int value(int c, int h) { return M::STEP * c + VAL * h; }
  __device__ void load_k(const void *base, int64_t at, int s, int slot, int h) {
    const T *p = (const T *)base + at + (int64_t)slot * DH;
#pragma unroll
    for (int c = 0; c < STEPS; ++c) kr[s][c] = *(const typename M::Op *)(p + value(c, h));
  }
  __device__ void load_v(const void *base, int64_t at, int slot, int r, int pr) {
    const T *p = (const T *)base + at + ((int64_t)r << pr) + slot;
#pragma unroll
    for (int i = 0; i < DH / 16; ++i) vr[i] = *(const typename M::Op *)(p + ((16 * i) << pr));
  }
  __device__ QOp k(int s, int c) const { return kr[s][c]; }
  static __device__ f4 mma(QOp a, QOp b, f4 c) { return M::mma(a, b, c); }
  static __device__ void q_parts(const float (&x)[VAL], QOp (&o)[PARTS]) {
    if constexpr (HALF) tree_q_halves(x, o[0], o[1]);
    else pa_parts<E>(x, o);
  }
  // the keys from the c-th on have no row behind them: nothing of what memory holds there
  __device__ void keep_v(int c) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (j >= c)
#pragma unroll
        for (int i = 0; i < DH / 16; ++i) vr[i][j] = (T)0.0f;
  }
  // the bits of values 16 i + r that are infinities or NaN, which are then cleared
  __device__ uint32_t take_odd(int i) {
    uint32_t odd = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (!__builtin_isfinite((float)vr[i][j])) odd |= 1u << j, vr[i][j] = (T)0.0f;
    return odd;
  }
  // how many keys both bits are set of
  static __device__ f4 count(uint32_t w, uint32_t v) {
    if constexpr (sizeof(T) == 2) {
      return tree_count(w, v, f4{0.0f, 0.0f, 0.0f, 0.0f});
    } else {
      typename M::Op a, b;
#pragma unroll
      for (int j = 0; j < PER; ++j) a[j] = w >> j & 1 ? 1.0f : 0.0f, b[j] = v >> j & 1 ? 1.0f : 0.0f;
      return M::mma(a, b, f4{0.0f, 0.0f, 0.0f, 0.0f});
    }
  }
  __device__ void add(const float (&p)[PER], f4 (&o)[DH / 16]) const {
    if constexpr (HALF) {
      PaTile<BF16>::Op pf[3], hi, lo;
      pa_parts<BF16>(p, pf);
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) pa_split(vr[i], hi, lo), o[i] = tree_split_mma(pf, hi, lo, o[i]);
    } else {
      pa_add<E>(p, vr, o);
    }
  }
};

template <class E, int DH>
struct TreeTile8 {
  using M = PaTile<F16>;
  using T = typename E::T;
  using QOp = M::Op;
  static constexpr bool SCALED = true, WIDE = true;
  static constexpr int KEYS = 64, SUB = 4, PER = 16, PARTS = 2, SUMS = 2, STEPS = DH / 32, VAL = 8;
  static constexpr float MOVE = 0x1p11f;
  static constexpr int HEAD = DH;
  u32x4 kr[SUB][(DH + 63) / 64], vr[DH / 16];
  // 16 bytes per lane are the values of two steps, 8 those of a last odd one
  static __device__ int value(int c, int h) {
    return c < DH / 64 * 2 ? 64 * (c / 2) + 16 * h + 8 * (c & 1) : 32 * c + 8 * h;
  }
  __device__ void load_k(const void *base, int64_t at, int s, int slot, int h) {
    const T *p = (const T *)base + at + (int64_t)slot * DH;
#pragma unroll
    for (int c = 0; c < DH / 64; ++c) kr[s][c] = *(const u32x4 *)(p + 64 * c + 16 * h);
    if (DH % 64) {
      const u32x2 x = *(const u32x2 *)(p + DH / 64 * 64 + 8 * h);
      kr[s][DH / 64] = u32x4{x[0], x[1], 0, 0};
    }
  }
  __device__ void load_v(const void *base, int64_t at, int slot, int r, int pr) {
    const T *p = (const T *)base + at + ((int64_t)r << pr) + slot;
#pragma unroll
    for (int i = 0; i < DH / 16; ++i) vr[i] = *(const u32x4 *)(p + ((16 * i) << pr));
  }
  __device__ QOp k(int s, int c) const {
    const u32x4 x = kr[s][c / 2];
    return Kv8<E>::f16(c & 1 ? u32x2{x[2], x[3]} : u32x2{x[0], x[1]});
  }
  static __device__ f4 mma(QOp a, QOp b, f4 c) { return M::mma(a, b, c); }
  static __device__ void q_parts(const float (&x)[VAL], QOp (&o)[PARTS]) {
    tree_q_halves(x, o[0], o[1]);
  }
  __device__ void keep_v(int c) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t mask = kv8_first(c - 4 * k);
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) vr[i][k] &= mask;
    }
  }
  __device__ uint32_t take_odd(int i) {
    uint32_t odd = 0;
    if (!Kv8<E>::FINITE)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t w = vr[i][k];
        odd |= kv8_take_nan(w) << (4 * k);
        vr[i][k] = w;
      }
    return odd;
  }
  static __device__ f4 count(uint32_t w, uint32_t v) {
    return tree_count(w >> 8, v >> 8, tree_count(w, v, f4{0.0f, 0.0f, 0.0f, 0.0f}));
  }
  __device__ void add(const float (&p)[PER], f4 (&o)[DH / 16]) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      PaTile<BF16>::Op pf[3];
      tree_parts(p + 8 * u, pf);
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) {
        const PaTile<BF16>::Op b = Kv8<E>::bf16(u ? u32x2{vr[i][2], vr[i][3]} : u32x2{vr[i][0], vr[i][1]});
#pragma unroll
        for (int k = 2; k >= 0; --k) o[i] = PaTile<BF16>::mma(pf[k], b, o[i]);
      }
    }
  }
};
template <int DH>
struct TreeTile<I8, DH> : TreeTile8<I8, DH> {};
template <int DH>
struct TreeTile<E4M3, DH> : TreeTile8<E4M3, DH> {};

// Turns over the keys: the weights at their own size; where means are not finite, at PA_LOW.  SCALED:
// before these, with the values' scales, and so the outputs, 2^40 times as large (see above).  (One row's scale of
// 2^100 passes the range then, also where its values are zeros and others' are not, which at PA_LOW would lose
// bits.  2^40 in the exponential's argument would cost no product, but the argument's own bits: 4.1e-7 off in
// place of 2.3e-7.)
constexpr float TREE_UP = 0x1p40f;
struct TreeTurn {
  float scale, up;  // of weights; of values' scales
  bool first;
};
template <bool SCALED>
__device__ inline TreeTurn tree_turn(int i) {
  if (SCALED) return TreeTurn{i < 2 ? 1.0f : PA_LOW, i == 0 ? TREE_UP : 1.0f, i == 0};
  return TreeTurn{i == 0 ? 1.0f : PA_LOW, 1.0f, i == 0};
}

// A query's running softmax (lane 16 h + r: query r) and its tile's output (lane
// 16 h + r: queries 4 h .., values 16 i + r).
template <bool SCALED, bool WIDE, int ND>
struct TreeSum {
  f4 o[ND];
  float m, sum;  // largest score, this lane's sum of weights
  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] = {};
    m = -__builtin_huge_valf(), sum = 0.0f;
  }
  // scores (c of them: log2; -inf: not seen) become the weights that enter the product with v
  template <int PER>
  __device__ __forceinline__ void weigh(float (&y)[PER], float c, const f4 *vsc, uint32_t sees, int h, float scale) {
    float top = y[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) top = fmaxf(top, y[j]);
    top *= c;
    if (__builtin_amdgcn_ballot_w64(top > m + PA_SLACK)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      // (each query's own: what others see changes no bit of it)
      const float next = top > m + PA_SLACK ? top : m, f = pa_weight(m, next);
      m = next;
      sum *= f;
      f4 fr;
#pragma unroll
      for (int i = 0; i < 4; ++i) fr[i] = __shfl(f, 4 * h + i);
#pragma unroll
      for (int i = 0; i < ND; ++i) o[i] *= fr;
    }
    const float base = m == -__builtin_huge_valf() ? 0.0f : m;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      y[j] = __builtin_amdgcn_exp2f(fmaf(y[j], c, -base));
      if (WIDE && scale != 1.0f) y[j] *= scale;
      sum += y[j];
      if constexpr (SCALED) y[j] = sees >> j & 1 ? y[j] * vsc[j >> 2][j & 3] : 0.0f;
    }
  }
  // values that are infinities or NaN and that not every query sees: NaN for those that do
  __device__ void spoil(int i, f4 seen) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (seen[e] > 0.0f) o[i][e] = __builtin_nanf("");
  }
  // what makes of a query's o its mean (0: it saw nothing); sum is then the query's
  __device__ float mean(float up) {
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    return sum == 0.0f ? 0.0f : 1.0f / (sum * up);
  }
};

// Query r's values in the scores' operand order; f16 parts: scaled by a power of two
// so that the largest lies in [2^14, 2^15), undone in the factor that is returned.  That power is 2^120
// at most, so that the factor (2^-120 times 0.13 and more) is no zero, which times an unseen
// key's -inf would be NaN: values below 2^-105 then lie lower, where a subnormal one, a multiple of
// 2^-149, still is the sum of its two parts, and a normal one, at 2^-6 at least, keeps 22 bits.
//   A key's scale may be as large as f32 goes.  So the part of that factor that makes smaller, and 2^-4
// more for the root of the head's size, is `low`, which the scale is multiplied by: a score that is in
// range in the end then is before the factor.  (Where low times a scale is no normal number
// and loses bits, the score is below 2^-93.)
template <class M, class T>
__device__ __forceinline__ float tree_q(const float *p, bool real, int h, T &qf, float &low) {
  float c = PA_LOG2E / __builtin_sqrtf((float)M::HEAD);
  low = 1.0f;
  float y[M::STEPS][M::VAL], top = 0.0f;
#pragma unroll
  for (int s = 0; s < M::STEPS; ++s)
#pragma unroll
    for (int j = 0; j < M::VAL; j += 4) {
      const f4 z = *(const f4 *)(p + M::value(s, h) + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[s][j + e] = real ? z[e] : 0.0f, top = fmaxf(top, __builtin_fabsf(y[s][j + e]));
    }
  int e = 0;
  if (M::MOVE != 1.0f) {
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    e = top > 0.0f ? max(__builtin_amdgcn_frexp_expf(top) - 15, -120) : 0;
    const int before = M::SCALED ? min(e - 4, 0) : 0;
    low = ldexpf(low, before);
    c = ldexpf(c, e - before);
  } else if (M::PARTS > 1) {
    e = pa_small(top), c = ldexpf(c, e);
  }
#pragma unroll
  for (int s = 0; s < M::STEPS; ++s) {
    typename M::QOp o[M::PARTS];
    if (M::PARTS > 1)
#pragma unroll
      for (int j = 0; j < M::VAL; ++j) y[s][j] = ldexpf(y[s][j], -e);
    M::q_parts(y[s], o);
#pragma unroll
    for (int k = 0; k < M::PARTS; ++k) qf[k][s] = o[k];
  }
  return c;
}

// One workgroup of PA_WAVES wavefronts per (tree, key/value head, 16 queries,
// chunk of keys).  A wavefront takes every PA_WAVES-th tile of keys, straight from memory, for
// all of the workgroup's queries.
// Bound, for long caches, by reading them: 61 rows of up to 8191 keys, 8 heads of 4 x 128, e4m3
// (390 MB) 103 us, 3.8 TB/s.  A wavefront has some 8 tiles of 64 keys to read, so that the first loads'
// way, the tile's chain (product, softmax, product) and the join are a quarter of it.  (8-bit heads
// of 128 need all registers and keep 14, e4m3, or 6, int8, of a lane's in memory.)  For short
// ones by that chain once: 6 heads of 64, 28 keys 6.4 us (int8), 114 keys 7.8 us (f32).
template <class E, int DH>
__global__ __launch_bounds__(64 * PA_WAVES, 2) void k_tree_attn(TreeArgs a) {
  using M = TreeTile<E, DH>;
  using QOp = typename M::QOp;
  constexpr int ND = DH / 16, KEYS = M::KEYS, PER = M::PER, SUB = M::SUB, PARTS = M::PARTS;
  constexpr int LD = DH + 4, NQ = 16;
  constexpr float NEG_INF = -__builtin_huge_valf();
  __shared__ float so[PA_WAVES][NQ][LD], sm[PA_WAVES][NQ], sl[PA_WAVES][NQ];

  // the query tiles of one (tree, head) run eight workgroups apart, on one XCD
  const int qi = blockIdx.x / 8 % a.qtiles, item = blockIdx.x / (8 * a.qtiles) * 8 + blockIdx.x % 8;
  const int hk = item % a.kv_heads, tree = item / a.kv_heads;
  if (tree >= a.n_trees) return;
  const TreeSpan sp = tree_span(a, tree);
  const int u0 = qi * NQ, all = sp.rows * a.group, nq = min(NQ, all - u0);
  if (nq <= 0) return;
  const int lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.kv_heads * a.group;
  const int n = tree_end(a, sp, u0 + nq);
  // query i of this workgroup: its row and head
  auto row_of = [&](int i) { return sp.start + (u0 + i) / a.group; };
  auto head_of = [&](int i) { return hk * a.group + (u0 + i) % a.group; };
  if (n <= 0) {
    if (blockIdx.y == 0)
      for (int i = threadIdx.x; i < nq * DH; i += 64 * PA_WAVES)
        a.out[row_of(i / DH) * a.ldo + (int64_t)head_of(i / DH) * DH + i % DH] = 0.0f;
    return;
  }
  const int k0 = blockIdx.y * a.chunk;
  if (k0 >= n) return;
  const bool direct = n <= a.chunk;
  const int end = (min(n, k0 + a.chunk) + KEYS - 1) / KEYS;
  const int P = 1 << a.pr;

  // The pages of this lane's k rows (keys PER (r / 4) on of a tile) and of its values (PER h
  // on).  Only read here: what is computed of them waits for them, and for the loads before them
  struct Where {
    int k, v;
  };
  auto where = [&](int t) __attribute__((always_inline)) {
    return Where{sp.table[min(t * KEYS + PER * (r >> 2), n - 1) >> a.pr], sp.table[min(t * KEYS + PER * h, n - 1) >> a.pr]};
  };
  auto in_pool = [&](int page) { return (unsigned)page < (unsigned)a.n_pages; };
  auto first = [&](int page) { return ((int64_t)(in_pool(page) ? page : 0) * a.kv_heads + hk) << a.pr; };  // row of the head
  M tile;
  f4 ksc[M::SCALED ? SUB : 1], vsc[M::SCALED ? SUB : 1];
  auto load_k = [&](int t, const Where &w) __attribute__((always_inline)) {
    const int64_t row = first(w.k);
#pragma unroll
    for (int s = 0; s < SUB; ++s) tile.load_k(a.k, row * DH, s, (t * KEYS + PER * (r >> 2) + 4 * s + (r & 3)) & (P - 1), h);
  };
  auto load_v = [&](int t, const Where &w) __attribute__((always_inline)) {
    const int slot = (t * KEYS + PER * h) & (P - 1);
    const int64_t row = first(w.v);
    tile.load_v(a.v, row * DH, slot, r, a.pr);
    if constexpr (M::SCALED)
#pragma unroll
      for (int s = 0; s < SUB; ++s) ksc[s] = *(const f4 *)(a.ks + row + slot + 4 * s), vsc[s] = *(const f4 *)(a.vs + row + slot + 4 * s);
  };

  const int t0 = k0 / KEYS + wv;
  int t = t0;
  Where now{}, next{};
  auto begin = [&]() __attribute__((always_inline)) {
    if (t < end) now = where(t), load_k(t, now);
    if (t + PA_WAVES < end) next = where(t + PA_WAVES);
  };
  begin();

  QOp qf[PARTS][M::STEPS];
  const int mine = min(r, nq - 1), node = (u0 + mine) / a.group;
  const uint32_t *mask = a.mask ? a.mask + (int64_t)row_of(mine) * a.n_words : nullptr;
  float low;
  const float c = tree_q<M>(a.q + row_of(mine) * a.ldq + (int64_t)head_of(mine) * DH, r < nq, h, qf, low);

  for (int i = 0;; ++i) {
    const TreeTurn turn = tree_turn<M::SCALED>(i);
    TreeSum<M::SCALED, M::WIDE, ND> acc;
    acc.clear();

    for (; t < end; t += PA_WAVES) {
      load_v(t, now);
      const bool more = t + PA_WAVES < end;
      f4 s[M::SUMS][SUB];
#pragma unroll
      for (int k = 0; k < M::SUMS; ++k)
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[k][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < M::STEPS; ++i)
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          const QOp kk = tile.k(u, i);
#pragma unroll
          for (int k = 0; k < PARTS; ++k) s[k % M::SUMS][u] = M::mma(kk, qf[k][i], s[k % M::SUMS][u]);
        }
      // (the pages of the tile after the next: they are there when its keys are asked for)
      Where after{};
      if (t + 2 * PA_WAVES < end) after = where(t + 2 * PA_WAVES);
      if (more) load_k(t + PA_WAVES, next);

      // keys that no query of the call may see, or that are in no page of the pool: no
      // weight, and what v holds there (anything) is taken as zero
      const int a0 = t * KEYS + PER * h;
      const bool bad = !in_pool(now.v);
      const bool edge = (t + 1) * KEYS > min(n, sp.past) || __builtin_amdgcn_ballot_w64(bad);
      bool odd_any = false;
      uint32_t odd[(ND + 1) / 2] = {};  // 16 bits for each i
      if (edge) {
        tile.keep_v(bad ? 0 : n - a0);
        // a row that one query sees and another does not may hold infinities or NaN:
        // they leave the products and are given to those who see them
#pragma unroll
        for (int i = 0; i < ND; ++i) odd[i / 2] |= tile.take_odd(i) << (16 * (i & 1));
#pragma unroll
        for (int i = 0; i < (ND + 1) / 2; ++i) odd_any |= odd[i] != 0;
        odd_any = __builtin_amdgcn_ballot_w64(odd_any) != 0;
      }
      float y[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        y[j] = s[M::SUMS - 1][j >> 2][j & 3];
#pragma unroll
        for (int k = M::SUMS - 2; k >= 0; --k) y[j] = fmaf(y[j], 1.0f / M::MOVE, s[k][j >> 2][j & 3]);
        if constexpr (M::SCALED) y[j] *= low * ksc[j >> 2][j & 3];
      }
      uint32_t sees = ~0u;
      if (edge) {
        sees = bad ? 0 : tree_sees<PER>(a, sp, mask, node, a0);
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (!(sees >> j & 1)) y[j] = NEG_INF;
      }
      if constexpr (M::SCALED)
#pragma unroll
        for (int u = 0; u < SUB; ++u) vsc[u] *= turn.up;
      acc.template weigh<PER>(y, c, vsc, sees, h, turn.scale);
      tile.add(y, acc.o);
      if (odd_any)
#pragma unroll
        for (int i = 0; i < ND; ++i) acc.spoil(i, M::count(sees, odd[i / 2] >> (16 * (i & 1))));
      now = next, next = after;
    }

    // the wavefront's means
    bool over = false;
    const float inv = acc.mean(turn.up);
    if (turn.first && h == 0) sm[wv][r] = acc.m, sl[wv][r] = acc.sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int qr = 4 * h + i;
      const float f = __shfl(inv, 4 * h + i);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const float y = acc.o[d][i] * f;
        float &mean = so[wv][qr][16 * d + r];
        if (!M::WIDE || turn.first) mean = y;
        else if (!__builtin_isfinite(mean)) mean = __builtin_isinf(y) && __builtin_isfinite(acc.o[d][i]) ? pa_largest(y) : y;
        over |= qr < nq && !__builtin_isfinite(y);
      }
    }
    if (!M::WIDE || turn.scale != 1.0f || !__builtin_amdgcn_ballot_w64(over)) break;
    t = t0;
    begin();
  }
  __syncthreads();

  // the wavefronts' means, each with its share of the weights
  const int64_t runs = (int64_t)a.rows * heads * gridDim.y;
  for (int i = threadIdx.x; i < nq * DH; i += 64 * PA_WAVES) {
    const int qr = i / DH, d = i % DH;
    float top = sm[0][qr], l = 0.0f, y = 0.0f, w[PA_WAVES];
#pragma unroll
    for (int k = 1; k < PA_WAVES; ++k) top = fmaxf(top, sm[k][qr]);
#pragma unroll
    for (int k = 0; k < PA_WAVES; ++k) l += w[k] = sl[k][qr] * pa_weight(sm[k][qr], top);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // 0: nothing is seen
#pragma unroll
    for (int k = 0; k < PA_WAVES; ++k) y += so[k][qr][d] * (w[k] * inv);
    if (M::WIDE && __builtin_isinf(y)) {
      bool finite = true;
#pragma unroll
      for (int k = 0; k < PA_WAVES; ++k) finite &= (bool)__builtin_isfinite(so[k][qr][d]);
      if (finite) y = pa_largest(y);
    }
    if (direct) {
      a.out[row_of(qr) * a.ldo + (int64_t)head_of(qr) * DH + d] = y;
    } else {
      const int64_t run = ((int64_t)row_of(qr) * heads + head_of(qr)) * gridDim.y + blockIdx.y;
      a.part[run * DH + d] = y;
      if (d == 0) a.part[runs * DH + 2 * run] = top, a.part[runs * DH + 2 * run + 1] = l;
    }
  }
}

// ------------------------------------------------- many queries of a tree
//
// The same with keys and values through LDS: the workgroup's wavefronts share a
// tile of them, each for 16 QW queries of its own, so that memory and L2 give a
// tile once for 64 QW queries and not once for 16.  What a wavefront reads
// of LDS are the operands themselves, 16 bytes a lane: K's rows lie in the order of
// the score product's rows, 8-bit values are converted and f16's v split where they are written,
// and the 16-byte units of a row are exchanged so that 16 lanes' reads fall into all banks.
//
// Bound by the matrix instructions and what must be done between them: with q and p in
// parts a bf16 pool takes 6 products of 16 x 16 x 32 where one of bf16 would take 2 (f16:
// 2 + 5, 8 bits: 2 + 3).  4 chunks of 512 rows behind 4100, 8 heads of 4 x 128, bf16: 439 us in a row of
// calls, 333 TFLOP/s of the formula's and 1000 of the products done; the matrix units are busy 40 % of the
// time, with two wavefronts to a SIMD of which each has some 250 other instructions to 48
// products.  (Straight from memory: 2.2 times that.  With the next tile's scores formed before this one's
// softmax: a tenth more.  With 128 queries: 557.)  The same chunks over int8: 468 us; 173 M vector instructions, where
// bf16 has 109 M, for the conversions and scales, 280 us of issue beside 146 of products.
// 24 trees of up to 48 rows, int8: 186 us, with half of the wavefronts' places empty, as the lengths are
// unlike: products are 29 us of it, vector instructions 61.

// units (16 bytes, 8 values) of a tile row of UNITS: where unit `col` of row `row` lies
template <int UNITS>
__device__ inline int tree_unit(int row, int col) {
  if constexpr (UNITS == 12) {
    const int c = col + (row >> 2 & 3);
    return row * 12 + (c >= 12 ? c - 12 : c);
  } else {
    return row * UNITS + (col ^ (row / (16 / UNITS) & (UNITS - 1)));
  }
}

template <class E, int DH>
struct TreeShared {
  using T = typename E::T;
  static constexpr bool SCALED = sizeof(T) == 1, HALF = std::is_same_v<E, F16>, WIDE = !HALF;
  using KE = std::conditional_t<std::is_same_v<E, BF16>, BF16, F16>;
  using M = PaTile<KE>;      // of the scores' product
  using W = PaTile<BF16>;    // of the second one
  using QOp = typename M::Op;
  static constexpr int PARTS = std::is_same_v<E, BF16> ? 3 : 2, SUMS = std::is_same_v<E, BF16> ? 1 : 2;
  static constexpr float MOVE = SUMS == 2 ? 0x1p11f : 1.0f;
  static constexpr int HEAD = DH, STEPS = DH / 32, VAL = 8;
  static constexpr int KEYS = SCALED || DH <= 64 ? 64 : 32;  // of a tile
  static constexpr int PLANES = HALF ? 2 : 1;                 // of v
  static constexpr int KU = DH / 8, VU = KEYS / 8;            // units of a row of K, of V
  static constexpr int RAW = 16 / sizeof(T);                  // values of 16 bytes of the pool
  static constexpr int LOADS = KEYS * DH / RAW;               // of 16 bytes, of K and of V each
  static constexpr int PER = (LOADS + 255) / 256;             // per thread
  static __device__ int value(int c, int h) { return 32 * c + 8 * h; }
  static __device__ void q_parts(const float (&x)[8], QOp (&o)[PARTS]) {
    if constexpr (SUMS == 2) tree_q_halves(x, o[0], o[1]);
    else pa_parts<BF16>(x, o);
  }
  struct Lds {  // a tile
    u32x4 k[KEYS * KU], v[PLANES][DH * VU];
    float ks[SCALED ? KEYS : 4], vs[SCALED ? KEYS : 4];
    unsigned long long odd[DH];  // keys whose value is an infinity or a NaN
  };
  // the row of K's tile that key `key` has: 16 s + 4 h + i for key 32 (s / 2) + 8 h + 4 (s % 2) + i
  static __device__ int k_row(int key) { return (key & 32) + (key >> 2 & 1) * 16 + (key >> 3 & 3) * 4 + (key & 3); }
};

template <class E, int DH, int QW, bool BIG>
__global__ __launch_bounds__(256, 2) void k_tree_shared(TreeArgs a) {
  using S = TreeShared<E, DH>;
  using T = typename E::T;
  constexpr int ND = DH / 16, KEYS = S::KEYS, PER = S::PER, PARTS = S::PARTS, SUMS = S::SUMS, RAW = S::RAW, NQ = 64 * QW;
  constexpr float NEG_INF = -__builtin_huge_valf();
  // One tile is computed with while the next is written; what is special about a tile (1: odd
  // values, 2: pages outside the pool) is cleared two tiles ahead
  __shared__ typename S::Lds lds[2];
  __shared__ int flags[3];

  const int qi = blockIdx.x / 8 % a.qtiles, item = blockIdx.x / (8 * a.qtiles) * 8 + blockIdx.x % 8;
  const int hk = item % a.kv_heads, tree = item / a.kv_heads;
  if (tree >= a.n_trees) return;
  const TreeSpan sp = tree_span(a, tree);
  const int u0 = qi * NQ, all = sp.rows * a.group, nq = min(NQ, all - u0);
  if (nq <= 0) return;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = a.kv_heads * a.group;
  const int n = tree_end(a, sp, u0 + nq);
  auto row_of = [&](int i) { return sp.start + (u0 + i) / a.group; };
  auto head_of = [&](int i) { return hk * a.group + (u0 + i) % a.group; };
  if (n <= 0) {
    if (blockIdx.y == 0)
      for (int i = tid; i < nq * DH; i += 256) a.out[row_of(i / DH) * a.ldo + (int64_t)head_of(i / DH) * DH + i % DH] = 0.0f;
    return;
  }
  const int k0 = blockIdx.y * a.chunk;
  if (k0 >= n) return;
  const bool direct = n <= a.chunk;
  const int t0 = k0 / KEYS, end = (min(n, k0 + a.chunk) + KEYS - 1) / KEYS, P = 1 << a.pr;
  // this wavefront's queries, and the end of what they see
  const int w0 = 16 * QW * wv, wq = min(16 * QW, nq - w0), wn = wq <= 0 ? 0 : tree_end(a, sp, u0 + w0 + wq);

  typename S::QOp qf[QW][PARTS][S::STEPS];
  float c[QW], low[QW];
  const uint32_t *mask[QW];
  int node[QW];
#pragma unroll
  for (int x = 0; x < QW; ++x) {
    const int i = min(w0 + 16 * x + r, nq - 1);
    node[x] = (u0 + i) / a.group;
    mask[x] = a.mask ? a.mask + (int64_t)row_of(i) * a.n_words : nullptr;
    c[x] = tree_q<S>(a.q + row_of(i) * a.ldq + (int64_t)head_of(i) * DH, w0 + 16 * x + r < nq, h, qf[x], low[x]);
  }

  // What this thread brings of a tile: 16 bytes of K's rows and of V's.  Pages no shorter
  // than a tile (BIG): its one page is the same for all threads, which add what is their
  // own for every tile; else each thread looks its pages up.
  u32x4 kr[PER], vr[PER];
  float kscale = 0.0f, vscale = 0.0f;
  int kp[BIG ? 1 : PER], vp[BIG ? 1 : PER], scale_page = 0;
  uint32_t vbad = 0;  // which of vr are of no page of the pool
  constexpr int KL = DH / RAW, VL = KEYS / RAW;  // loads of a row of K, of V
  auto key_of = [&](int i) { return (i * 256 + tid) / KL; };
  auto group_of = [&](int i) { return (i * 256 + tid) % VL * RAW; };  // first key
  auto page_of = [&](int key) { return sp.table[min(key, n - 1) >> a.pr]; };
  auto in_pool = [&](int page) { return (unsigned)page < (unsigned)a.n_pages; };
  auto first = [&](int page) { return ((int64_t)(in_pool(page) ? page : 0) * a.kv_heads + hk) << a.pr; };
  auto pages = [&](int t) __attribute__((always_inline)) {
    if constexpr (BIG) {
      // (a scalar load: a vector load's result would be waited for together with the tile's own, which are behind it)
      typedef const __attribute__((address_space(4))) int32_t *Scalar;
      kp[0] = ((Scalar)(uintptr_t)sp.table)[__builtin_amdgcn_readfirstlane(min(t * KEYS, n - 1) >> a.pr)];
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) kp[i] = page_of(t * KEYS + min(key_of(i), KEYS - 1)), vp[i] = page_of(t * KEYS + group_of(i));
      if (S::SCALED && tid < KEYS) scale_page = page_of(t * KEYS + tid);
    }
  };
  auto load = [&](int t) __attribute__((always_inline)) {
    vbad = 0;
    const int64_t one = BIG ? first(kp[0]) : 0;
    const int at = t * KEYS & (P - 1);
    const char *kb = (const char *)a.k + (one + at) * (DH * (int)sizeof(T)), *vb = (const char *)a.v + (one * DH + at) * (int)sizeof(T);
    if (BIG && !in_pool(kp[0])) vbad = ~0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 256 + tid;
      if (S::LOADS % 256 && e >= S::LOADS) break;
      if constexpr (BIG) {
        kr[i] = *(const u32x4 *)(kb + (uint32_t)e * 16);
        vr[i] = *(const u32x4 *)(vb + (((uint32_t)(e / VL) << a.pr) * (uint32_t)sizeof(T) + (uint32_t)(e % VL) * 16));
      } else {
        vbad |= in_pool(vp[i]) ? 0u : 1u << i;
        kr[i] = *(const u32x4 *)((const T *)a.k + (first(kp[i]) + ((t * KEYS + key_of(i)) & (P - 1))) * DH + e % KL * RAW);
        vr[i] = *(const u32x4 *)((const T *)a.v + first(vp[i]) * DH + ((int64_t)(e / VL) << a.pr) + ((t * KEYS + group_of(i)) & (P - 1)));
      }
    }
    if (S::SCALED && tid < KEYS) {
      const int64_t row = BIG ? one + at + tid : first(scale_page) + ((t * KEYS + tid) & (P - 1));
      kscale = a.ks[row], vscale = a.vs[row];
    }
  };
  TreeTurn turn;
  // ... goes to LDS
  auto store = [&](int t, bool edge) __attribute__((always_inline)) {
    typename S::Lds &l = lds[t & 1];
    auto put = [&](int i, u32x4 y) __attribute__((always_inline)) {
      const int e = i * 256 + tid, krow = S::k_row(key_of(i)), kc = e % KL, value = e / VL, vc = e % VL;
      if constexpr (S::SCALED) {
        const u32x4 x = kr[i];
        l.k[tree_unit<S::KU>(krow, 2 * kc)] = __builtin_bit_cast(u32x4, Kv8<E>::f16(u32x2{x[0], x[1]}));
        l.k[tree_unit<S::KU>(krow, 2 * kc + 1)] = __builtin_bit_cast(u32x4, Kv8<E>::f16(u32x2{x[2], x[3]}));
        l.v[0][tree_unit<S::VU>(value, 2 * vc)] = __builtin_bit_cast(u32x4, Kv8<E>::bf16(u32x2{y[0], y[1]}));
        l.v[0][tree_unit<S::VU>(value, 2 * vc + 1)] = __builtin_bit_cast(u32x4, Kv8<E>::bf16(u32x2{y[2], y[3]}));
      } else {
        l.k[tree_unit<S::KU>(krow, kc)] = kr[i];
        if constexpr (S::HALF) {
          typename S::W::Op hi, lo;
          pa_split(__builtin_bit_cast(PaTile<F16>::Op, y), hi, lo);
          l.v[0][tree_unit<S::VU>(value, vc)] = __builtin_bit_cast(u32x4, hi);
          l.v[1][tree_unit<S::VU>(value, vc)] = __builtin_bit_cast(u32x4, lo);
        } else {
          l.v[0][tree_unit<S::VU>(value, vc)] = y;
        }
      }
    };
    if (S::SCALED && tid < KEYS) l.ks[tid] = kscale, l.vs[tid] = vscale * turn.up;
    if (!edge && !__builtin_amdgcn_ballot_w64(vbad != 0)) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (S::LOADS % 256 && i * 256 + tid >= S::LOADS) break;
        put(i, vr[i]);
      }
      return;
    }
    // v behind the rows and in pages that are not there (anything): zeros.  At an edge, where a row that one
    // query sees and another does not may hold infinities or NaN, these leave the products and are given to
    // those who see them.  Another tile of which pages are not there keeps what the others hold, which all
    // queries see (BIG: it has no others)
    const bool take = BIG || edge;
    int special = vbad ? 2 : 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 256 + tid;
      if (S::LOADS % 256 && e >= S::LOADS) break;
      const int vc = e % VL, have = vbad >> i & 1 ? 0 : n - (t * KEYS + vc * RAW);  // keys with a row behind them
      u32x4 y = vr[i];
      uint32_t odd = 0;
      if constexpr (S::SCALED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w = y[j] & kv8_first(have - 4 * j);
          if (!Kv8<E>::FINITE && take) odd |= kv8_take_nan(w) << (4 * j);
          y[j] = w;
        }
      } else {
        typename PaTile<E>::Op z = __builtin_bit_cast(typename PaTile<E>::Op, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= have) z[j] = (T)0.0f;
          if (take && !__builtin_isfinite((float)z[j])) odd |= 1u << j, z[j] = (T)0.0f;
        }
        y = __builtin_bit_cast(u32x4, z);
      }
      put(i, y);
      if (odd && edge) atomicOr(&l.odd[e / VL], (unsigned long long)odd << (vc * RAW)), special |= 1;
    }
    if (special) atomicOr(&flags[t % 3], special);
  };

  for (int i = 0;; ++i) {
    turn = tree_turn<S::SCALED>(i);
    TreeSum<S::SCALED, S::WIDE, ND> acc[QW];
#pragma unroll
    for (int x = 0; x < QW; ++x) acc[x].clear();
    auto edge_of = [&](int t) { return (t + 1) * KEYS > min(n, sp.past); };
    auto clear_odd = [&](int t) __attribute__((always_inline)) {
      if (tid < DH) lds[t & 1].odd[tid] = 0;
      __syncthreads();
    };
    pages(t0);
    load(t0);
    if (t0 + 1 < end) pages(t0 + 1);
    __syncthreads();  // (a second time: the first is done)
    if (tid < 3) flags[tid] = 0;
    clear_odd(t0);
    store(t0, edge_of(t0));

    for (int t = t0; t < end; ++t) {
      __syncthreads();  // tile t is there, and t - 1 is done with
      const bool edge = edge_of(t), more = t + 1 < end;
      if (more) {
        load(t + 1);
        if (t + 2 < end) pages(t + 2);
      }
      if (tid == 0) flags[(t + 2) % 3] = 0;
      const typename S::Lds &l = lds[t & 1];
      if (t * KEYS < wn) {
        const int special = flags[t % 3];
        const bool odd_any = special & 1, bad_any = special & 2;
#pragma unroll
        for (int u = 0; u < KEYS / 32; ++u) {
          f4 s[QW][SUMS][2];
#pragma unroll
          for (int x = 0; x < QW; ++x)
#pragma unroll
            for (int k = 0; k < SUMS; ++k) s[x][k][0] = s[x][k][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < S::STEPS; ++i)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const auto kk = __builtin_bit_cast(typename S::QOp, l.k[tree_unit<S::KU>(32 * u + 16 * b + r, 4 * i + h)]);
#pragma unroll
              for (int x = 0; x < QW; ++x)
#pragma unroll
                for (int k = 0; k < PARTS; ++k) s[x][k % SUMS][b] = S::M::mma(kk, qf[x][k][i], s[x][k % SUMS][b]);
            }
          const int a0 = t * KEYS + 32 * u + 8 * h;
          f4 ksc[2], vsc[2];
          if constexpr (S::SCALED)
#pragma unroll
            for (int b = 0; b < 2; ++b) ksc[b] = *(const f4 *)&l.ks[32 * u + 8 * h + 4 * b], vsc[b] = *(const f4 *)&l.vs[32 * u + 8 * h + 4 * b];
          uint32_t there = 0xFF;
          if (bad_any && !in_pool(page_of(a0))) there = 0;
          typename S::W::Op pf[QW][3];
          uint32_t sees[QW];
#pragma unroll
          for (int x = 0; x < QW; ++x) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              y[j] = s[x][SUMS - 1][j >> 2][j & 3];
              if (SUMS == 2) y[j] = fmaf(y[j], 1.0f / S::MOVE, s[x][0][j >> 2][j & 3]);
              if constexpr (S::SCALED) y[j] *= low[x] * ksc[j >> 2][j & 3];
            }
            sees[x] = 0xFF;
            if (edge || bad_any) {
              sees[x] = there & tree_sees<8>(a, sp, mask[x], node[x], a0);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (!(sees[x] >> j & 1)) y[j] = NEG_INF;
            }
            acc[x].template weigh<8>(y, c[x], vsc, sees[x], h, turn.scale);
            pa_parts<BF16>(y, pf[x]);
          }
          // (two outputs in turn: a matrix instruction waits for the one before it on the same)
#pragma unroll
          for (int i = 0; i < ND; i += 2) {
            typename S::W::Op v[S::PLANES][2];
#pragma unroll
            for (int p = 0; p < S::PLANES; ++p)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                v[p][e] = __builtin_bit_cast(typename S::W::Op, l.v[p][tree_unit<S::VU>(16 * (i + e) + r, 4 * u + h)]);
            // parts of p (2: least) and of v (1: less)
            auto add = [&](int k, int p) __attribute__((always_inline)) {
#pragma unroll
              for (int x = 0; x < QW; ++x)
#pragma unroll
                for (int e = 0; e < 2; ++e) acc[x].o[i + e] = S::W::mma(pf[x][k], v[p][e], acc[x].o[i + e]);
            };
            add(2, 0);
            if (S::HALF) add(1, S::PLANES - 1);
            add(1, 0);
            if (S::HALF) add(0, S::PLANES - 1);
            add(0, 0);
          }
          if (odd_any && edge)
#pragma unroll
            for (int i = 0; i < ND; ++i) {
              const uint32_t odd = (uint32_t)(l.odd[16 * i + r] >> (32 * u + 8 * h)) & 0xFF;
#pragma unroll
              for (int x = 0; x < QW; ++x) acc[x].spoil(i, tree_count(sees[x], odd, f4{0.0f, 0.0f, 0.0f, 0.0f}));
            }
        }
      }
      if (more) {
        if (edge_of(t + 1)) clear_odd(t + 1);
        store(t + 1, edge_of(t + 1));
      }
    }

    // the means, to where they go (a second time: where the first ones are not finite)
    const bool again = !turn.first;
    bool over = false;
    const int64_t runs = (int64_t)a.rows * heads * gridDim.y;
#pragma unroll
    for (int x = 0; x < QW; ++x) {
      const float inv = acc[x].mean(turn.up);
      const int mine = w0 + 16 * x + r;
      if (!direct && !again && h == 0 && mine < nq) {
        const int64_t run = ((int64_t)row_of(mine) * heads + head_of(mine)) * gridDim.y + blockIdx.y;
        a.part[runs * DH + 2 * run] = acc[x].m, a.part[runs * DH + 2 * run + 1] = acc[x].sum;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int qr = w0 + 16 * x + 4 * h + i;
        const float f = __shfl(inv, 4 * h + i);
        if (qr >= nq) continue;
        float *dst = direct ? a.out + row_of(qr) * a.ldo + (int64_t)head_of(qr) * DH
                            : a.part + (((int64_t)row_of(qr) * heads + head_of(qr)) * gridDim.y + blockIdx.y) * DH;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const float y = acc[x].o[d][i] * f;
          if (!again) dst[16 * d + r] = y;
          else if (!__builtin_isfinite(dst[16 * d + r]))
            dst[16 * d + r] = __builtin_isinf(y) && __builtin_isfinite(acc[x].o[d][i]) ? pa_largest(y) : y;
          over |= !__builtin_isfinite(y);
        }
      }
    }
    if (!S::WIDE || turn.scale != 1.0f || !__syncthreads_or(over)) break;
  }
}

// The chunks of one query, joined as k_paged_join joins them.  blockIdx.x = (tree x
// max_rows + row of the tree) x heads + head; nq: queries per workgroup of k_tree_attn.
template <int DH>
__global__ __launch_bounds__(256) void k_tree_join(TreeArgs a, int nsplit, int nq) {
  constexpr int W = DH <= 32 ? 8 : DH <= 64 ? 16 : 32, SIDE = 256 / W;  // W threads of 4 values
  __shared__ float sw[PA_MAX_SPLIT], sl[4];
  __shared__ f4 sy[SIDE][DH / 4];
  const int heads = a.kv_heads * a.group, most = a.starts ? a.max_rows : 1;
  const int hq = blockIdx.x % heads, tree = blockIdx.x / heads / most, j = blockIdx.x / heads % most;
  const TreeSpan sp = tree_span(a, tree);
  if (j >= sp.rows) return;
  const int u = j * a.group + hq % a.group;
  const int n = tree_end(a, sp, min(u / nq * nq + nq, sp.rows * a.group));
  if (n <= a.chunk) return;
  const int nz = (n + a.chunk - 1) / a.chunk;  // <= nsplit <= PA_MAX_SPLIT
  const int64_t row = sp.start + j, run0 = (row * heads + hq) * nsplit, runs = (int64_t)a.rows * heads * nsplit;
  const float *ml = a.part + runs * DH + 2 * run0;
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
    const f4 *o = (const f4 *)(a.part + run0 * DH) + d;
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
      for (int z = 0; z < nz; ++z) finite &= (bool)__builtin_isfinite(a.part[(run0 + z) * DH + threadIdx.x]);
      if (finite) y = pa_largest(y);
    }
    a.out[row * a.ldo + (int64_t)hq * DH + threadIdx.x] = y;
  }
}

// The same for up to JOIN_FEW chunks: a wavefront a query, a lane a chunk's weight.
// (24 trees of 48 rows, 32 heads of 128, 3 chunks: 11.6 us, by a workgroup a query 29.9; 61 rows, 4 chunks: 5.3 and 5.4)
constexpr int JOIN_FEW = 64;
template <int DH>
__global__ __launch_bounds__(256) void k_tree_join_few(TreeArgs a, int nsplit, int nq, int queries) {
  const int heads = a.kv_heads * a.group, most = a.starts ? a.max_rows : 1;
  const int i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= queries) return;
  const int hq = i % heads, tree = i / heads / most, j = i / heads % most;
  const TreeSpan sp = tree_span(a, tree);
  if (j >= sp.rows) return;
  const int u = j * a.group + hq % a.group;
  const int n = tree_end(a, sp, min(u / nq * nq + nq, sp.rows * a.group));
  if (n <= a.chunk) return;
  const int nz = (n + a.chunk - 1) / a.chunk;
  const int64_t row = sp.start + j, run0 = (row * heads + hq) * nsplit, runs = (int64_t)a.rows * heads * nsplit;
  const float *ml = a.part + runs * DH + 2 * run0, *o = a.part + run0 * DH;
  const float m = lane < nz ? ml[2 * lane] : -__builtin_huge_valf(), l = lane < nz ? ml[2 * lane + 1] : 0.0f;
  float top = m;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
  const float w = l * pa_weight(m, top);
  float total = w;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) total += __shfl_xor(total, x);
  const float share = total == 0.0f ? 0.0f : w * (1.0f / total);
  constexpr int V = (DH + 63) / 64;
  float y[V] = {};
  bool finite[V];
#pragma unroll
  for (int d = 0; d < V; ++d) finite[d] = true;
  for (int z0 = 0; z0 < nz; z0 += 4)
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // (four loads on their way; behind the last chunk: it again, of no weight)
      const int z = min(z0 + e, nz - 1);
      const float s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(share), z)), f = z0 + e < nz ? s : 0.0f;
#pragma unroll
      for (int d = 0; d < V; ++d)
        if (DH % 64 == 0 || 64 * d + lane < DH) {
          const float x = o[z * DH + 64 * d + lane];
          y[d] += x * f;
          finite[d] &= (bool)__builtin_isfinite(x);
        }
    }
#pragma unroll
  for (int d = 0; d < V; ++d)
    if (DH % 64 == 0 || 64 * d + lane < DH)
      a.out[row * a.ldo + (int64_t)hq * DH + 64 * d + lane] = __builtin_isinf(y[d]) && finite[d] ? pa_largest(y[d]) : y[d];
}

#endif  // __HIPCC__

}  // namespace rw
