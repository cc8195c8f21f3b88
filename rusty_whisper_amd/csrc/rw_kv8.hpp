// rw_kv8.hpp -- pages of 8 bits: rows quantised as they are written; and rows of
// any pool read back.
//
// A row of one head has one scale, s = max(amax / TOP, 2^-126) in f32 (TOP: 127
// for whole numbers, 448 for e4m3), and every value is the nearest that the type
// has to x / s, so it reads back within s / 2 (i8) or 2^-4 of itself (e4m3, s 2^-10
// where that is larger).  The quotient is formed in 64 bits, correctly rounded,
// so that no rounding but the last decides between two neighbours.  A row that
// holds an infinity or a NaN has the scale NaN and zeros: it reads back as NaN.
#pragma once
#include "rw_kv.hpp"

namespace rw {

#if defined(__HIPCC__)

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 8-bit pools' types; code4: of four scaled values x / s
struct I8 {
  using T = int8_t;
  static constexpr float TOP = 127.0f;
  static __device__ float load(const T *p) { return (float)*p; }
  static __device__ uint32_t code4(const double (&y)[4]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)__builtin_rint(y[i]) & 0xFF) << (8 * i);
    return w;
  }
};
struct E4M3 {
  using T = uint8_t;
  static constexpr float TOP = 448.0f;
  static __device__ float load(const T *p) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 y = __builtin_amdgcn_cvt_pk_f32_fp8((int)*p, false);
    return y[0];
  }
  // y to 24 bits, the last one set where bits are lost, so that the rounding to
  // the type's 4 bits sees on which side of a middle y lies
  static __device__ float sticky(double y) {
    uint64_t b = __builtin_bit_cast(uint64_t, y);
    b = (b & ~(uint64_t)0x1FFFFFFF) | ((b & 0x1FFFFFFF) != 0 ? (uint64_t)0x20000000 : 0);
    return (float)__builtin_bit_cast(double, b);
  }
  static __device__ uint32_t code4(const double (&y)[4]) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(sticky(y[0]), sticky(y[1]), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(sticky(y[2]), sticky(y[3]), w, true);
  }
};

// the scale of a row whose largest magnitude has the bits `amax`
template <class E>
__device__ inline float kv8_scale(uint32_t amax) {
  return amax >= 0x7F800000u ? __builtin_nanf("") : fmaxf(__uint_as_float(amax) / E::TOP, 0x1p-126f);
}
// the codes of 8 values: with inv = 1 / s rounded once, one step of correction
// makes the quotient in 64 bits the correctly rounded one
template <class E>
__device__ inline uint2 kv8_codes(const float (&x)[8], float s) {
  if (!(s == s)) return make_uint2(0, 0);
  const double d = s, inv = 1.0 / d;
  uint2 w;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    double y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double a = x[4 * p + i], q = a * inv;
      y[i] = __builtin_copysign(__builtin_fma(__builtin_fma(-q, d, a), inv, q), a);
    }
    (p ? w.y : w.x) = E::code4(y);
  }
  return w;
}

// where row r of a call goes: the page (-1: no place) and the row in it
__device__ inline int kv_place(const PagedView &w, int r, int p, int *slot) {
  const int32_t *table = paged_row(w, r);
  *slot = p & ((1 << w.pr) - 1);
  if (!table || p < 0 || (p >> w.pr) >= w.ld) return -1;
  const int page = table[p >> w.pr];
  return (unsigned)page < (unsigned)w.n_pages ? page : -1;
}

// K8_ROWS rows of one head per workgroup, 8 values of k and of v per thread and
// turn.  A row's threads are neighbouring lanes, which find its largest value by
// exchanges; v's codes cross through LDS and go out four rows at a time where four rows
// of a page follow each other.  Bound by memory: 36000 rows of 20 heads of 64, e4m3 (460 MB), 133
// us, 3.5 TB/s; 64 rows, int8: 6.8 us (64 rows per workgroup: 133 and 9.6).
constexpr int K8_ROWS = 32;
template <class E, int DH>
__global__ __launch_bounds__(256) void k_kv_write8(PagedView w, const float *__restrict__ k, int64_t ldk,
                                                   const float *__restrict__ v, int64_t ldv, int rows,
                                                   const int32_t *__restrict__ pos, int tiles, int row0) {
  constexpr int LANES = DH <= 32 ? 4 : DH <= 64 ? 8 : 16;  // of a row; DH / 8 of them have values
  __shared__ uint8_t sv[K8_ROWS][DH + 4];
  __shared__ int page[K8_ROWS], slot[K8_ROWS];
  const int tile = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);  // gridDim.x: a multiple of 8
  if (tile >= tiles) return;
  const int t = threadIdx.x, head = tile % w.heads, r0 = row0 + tile / w.heads * K8_ROWS;
  if (t < K8_ROWS) {
    int at = -1, sl = 0;
    if (r0 + t < rows) at = kv_place(w, r0 + t, pos[r0 + t], &sl);
    page[t] = at, slot[t] = sl;
  }
  __syncthreads();
  const int64_t per = (int64_t)DH << w.pr;  // a page's values of one head
#pragma unroll
  for (int i0 = 0; i0 < K8_ROWS; i0 += 256 / LANES) {
    const int i = i0 + t / LANES, d = t % LANES * 8;
    if (256 / LANES > K8_ROWS && i >= K8_ROWS) break;
    const bool in = r0 + i < rows && d < DH;
    float x[2][8];
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float *a = (p ? v + (int64_t)(r0 + i) * ldv : k + (int64_t)(r0 + i) * ldk) + head * DH + d;
      const f4 a0 = in ? *(const f4 *)a : f4{0, 0, 0, 0}, a1 = in ? *(const f4 *)(a + 4) : f4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[p][j] = j < 4 ? a0[j] : a1[j - 4];
        top[p] = max(top[p], __float_as_uint(x[p][j]) & 0x7FFFFFFFu);
      }
    }
#pragma unroll
    for (int s = 1; s < LANES; s <<= 1) {
      top[0] = max(top[0], (uint32_t)__shfl_xor((int)top[0], s));
      top[1] = max(top[1], (uint32_t)__shfl_xor((int)top[1], s));
    }
    const float sk = kv8_scale<E>(top[0]), sv_ = kv8_scale<E>(top[1]);
    if (!in) continue;
    const uint2 ck = kv8_codes<E>(x[0], sk), cv = kv8_codes<E>(x[1], sv_);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sv[i][d + j] = (uint8_t)(cv.x >> (8 * j));
      sv[i][d + 4 + j] = (uint8_t)(cv.y >> (8 * j));
    }
    if (page[i] >= 0) {
      const int64_t at = (int64_t)page[i] * w.heads + head;
      *(uint2 *)((uint8_t *)w.k + at * per + (int64_t)slot[i] * DH + d) = ck;
      if (d == 0) w.ks[(at << w.pr) + slot[i]] = sk, w.vs[(at << w.pr) + slot[i]] = sv_;
    }
  }
  __syncthreads();
  // rows four by four, from the first that begins a group of four in its page on (a
  // group before it and one behind are short)
  const int shift = -slot[0] & 3;
  constexpr int GROUPS = K8_ROWS / 4 + 1;
  for (int e = t; e < GROUPS * DH; e += 256) {
    const int g = e % GROUPS, d = e / GROUPS, i0 = shift - 4 + 4 * g;
    bool four = i0 >= 0 && i0 + 3 < K8_ROWS && (slot[i0 < 0 ? 0 : i0] & 3) == 0;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j;
      if (i < 0 || i >= K8_ROWS || page[i] < 0) {
        four = false;
        continue;
      }
      if (four) four = page[i] == page[i0] && slot[i] == slot[i0] + j;
      word |= (uint32_t)sv[i][d] << (8 * j);
    }
    uint8_t *base = (uint8_t *)w.v + (int64_t)head * per + ((int64_t)d << w.pr);
    if (four) {
      *(uint32_t *)(base + (int64_t)page[i0] * w.heads * per + slot[i0]) = word;
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j;
      if (i >= 0 && i < K8_ROWS && page[i] >= 0) base[(int64_t)page[i] * w.heads * per + slot[i]] = (uint8_t)(word >> (8 * j));
    }
  }
}

// Rows of pages as f32: ROWS rows of one head per workgroup, values as they are
// stored through LDS.  v's rows are innermost in a page: its words hold GROUP rows of
// one value, and are read whole where rows follow each other.  A row without a place
// reads as zeros.
// Bound by three trips to memory in a row (position, page, values) and the writes: 36000
// rows of 20 heads of 64, e4m3 (460 MB), 130 us with ROWS = 64, 152 with 32 (197 by single values of
// v); 64 rows, int8: 8.0 us with 64, 6.3 with 32.
template <class E, int DH, int ROWS>
__global__ __launch_bounds__(256) void k_kv_read(PagedView w, float *__restrict__ k, int64_t ldk, float *__restrict__ v,
                                                 int64_t ldv, int rows, const int32_t *__restrict__ pos, int tiles, int row0) {
  using T = typename E::T;
  typedef T In __attribute__((ext_vector_type(8)));
  constexpr int LANES = DH <= 32 ? 4 : DH <= 64 ? 8 : 16;  // of a row; DH / 8 of them have values
  constexpr int STEP = 256 / LANES, PASSES = ROWS / STEP > 1 ? ROWS / STEP : 1;
  constexpr int GROUP = 4 / sizeof(T), GROUPS = ROWS / GROUP + (GROUP > 1), WORDS = (GROUPS * DH + 255) / 256;
  __shared__ alignas(16) T sv[ROWS][DH + 16 / sizeof(T)];
  __shared__ int page[ROWS], slot[ROWS], whole[GROUPS];  // whole: the page of a group's rows, -1: one by one
  __shared__ float scale[2][ROWS];
  const int tile = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);  // gridDim.x: a multiple of 8
  if (tile >= tiles) return;
  const int t = threadIdx.x, head = tile % w.heads, r0 = row0 + tile / w.heads * ROWS;
  if (t < ROWS) {
    int at = -1, sl = 0;
    if (r0 + t < rows) at = kv_place(w, r0 + t, pos[r0 + t], &sl);
    page[t] = at, slot[t] = sl;
  }
  __syncthreads();
  // groups of rows from the first that begins one in its page on (one before it and one behind are short)
  const int shift = GROUP == 1 ? 0 : (-slot[0] & (GROUP - 1)) - GROUP;
  if (t < GROUPS) {
    const int i0 = shift + GROUP * t;
    int at = -1;
    if (i0 >= 0 && i0 + GROUP <= ROWS && (slot[i0] & (GROUP - 1)) == 0) {
      at = page[i0];
      for (int j = 1; j < GROUP; ++j) at = page[i0 + j] == at && slot[i0 + j] == slot[i0] + j ? at : -1;
    }
    whole[t] = at;
  }
  if (w.ks && t >= 64 && t < 64 + 2 * ROWS) {
    const int i = t % ROWS, side = (t - 64) / ROWS;
    scale[side][i] = page[i] < 0 ? 1.0f : (side ? w.vs : w.ks)[(((int64_t)page[i] * w.heads + head) << w.pr) + slot[i]];
  }
  __syncthreads();

  // all loads on their way before the first is waited for
  const int d = t % LANES * 8;
  In a[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int i = min(p * STEP + t / LANES, ROWS - 1);
    const int64_t row = (((int64_t)max(page[i], 0) * w.heads + head) << w.pr) + slot[i];
    a[p] = *(const In *)((const T *)w.k + row * DH + min(d, DH - 8));
  }
  auto v_at = [&](int at, int value) { return (const T *)w.v + ((((int64_t)at * w.heads + head) * DH + value) << w.pr); };
  uint32_t word[WORDS];
#pragma unroll
  for (int x = 0; x < WORDS; ++x) {
    const int e = min(x * 256 + t, GROUPS * DH - 1), g = e % GROUPS, at = whole[g];
    word[x] = *(const uint32_t *)(v_at(max(at, 0), e / GROUPS) + (at < 0 ? 0 : slot[shift + GROUP * g]));
  }
#pragma unroll
  for (int x = 0; x < WORDS; ++x) {
    const int e = x * 256 + t, g = e % GROUPS, value = e / GROUPS, i0 = shift + GROUP * g;
    if (e >= GROUPS * DH) break;
    T y[GROUP];
    __builtin_memcpy(y, &word[x], 4);
    if (whole[g] < 0)
#pragma unroll
      for (int j = 0; j < GROUP; ++j) {
        const int i = i0 + j;
        y[j] = i >= 0 && i < ROWS && page[i] >= 0 ? v_at(page[i], value)[slot[i]] : (T)0;
      }
#pragma unroll
    for (int j = 0; j < GROUP; ++j)
      if (GROUP == 1 || (i0 + j >= 0 && i0 + j < ROWS)) sv[i0 + j][value] = y[j];
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int i = p * STEP + t / LANES;
    if (i >= ROWS || r0 + i >= rows || d >= DH) continue;
    const In b = *(const In *)&sv[i][d];
    const bool have = page[i] >= 0;
    f4 y[2][2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const T xk = a[p][j], xv = b[j];
      y[0][j >> 2][j & 3] = have ? E::load(&xk) : 0.0f, y[1][j >> 2][j & 3] = E::load(&xv);
    }
    if (w.ks) {
      const float sk = scale[0][i], sx = scale[1][i];
#pragma unroll
      for (int h = 0; h < 2; ++h) y[0][h] *= sk, y[1][h] *= sx;
    }
    float *ok = k + (int64_t)(r0 + i) * ldk + head * DH + d, *ov = v + (int64_t)(r0 + i) * ldv + head * DH + d;
    *(f4 *)ok = y[0][0], *(f4 *)(ok + 4) = y[0][1];
    *(f4 *)ov = y[1][0], *(f4 *)(ov + 4) = y[1][1];
  }
}

#endif  // __HIPCC__

}  // namespace rw
