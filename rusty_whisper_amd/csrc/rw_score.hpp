// rw_score.hpp -- log-probs of given tokens, entropy and top alternatives of
// rows of logits.
//
// With M = max x, S = sum e^(x - M), T = sum (x - M) e^(x - M):
//   lp(t) = x_t - M - ln S,   entropy = ln S - T / S
// (both terms of the entropy are non-negative, so nothing cancels).
//
// k_score reads its part of a row once, in steps of 64 x PER logits per
// wavefront, which stay in registers while the step's maximum, sums and
// candidates are formed.  A lane keeps M, S and T of its own logits (raised
// maxima scale S and T); lanes, wavefronts and parts are joined at the end in
// a fixed order.
//
// The alternatives.  `lo` is the smallest logit that may be one of the k best: of
// the k best so far, kept one per lane, the next above the k-th (later ids are
// larger, so an equal logit comes too late), or the k-th largest of the lanes'
// maxima so far, which score_bound finds to within a few.  Most steps end with
// one comparison; the logits from lo on are collected in LDS, and from time to
// time (for few alternatives in every step) they are put into the k best: a few
// one by one, more of them ranked, an entry's rank being the number of entries
// before it (larger, or equal with a smaller id).  366 rows of 51865 f32 with 20
// alternatives: 28 to 31 us; ranked in every step 35; with 5, every step 22.
//
// Bound by reading the logits: 1792 rows of 51866 f32, 372 MB, 68 us without
// alternatives (5.4 TB/s), 71 with 5, 77 to 80 with 16, 100 to 108 with 32; f16 45
// and 58 to 68 (4.1 TB/s: the exponentials and the conversion begin to show).
// Rows whose logits rise with their ids take longest (every step replaces the k
// best: 204 us with 5).  One row: latency, 4.6 us with 5 alternatives and 3.8 for
// the join.
#pragma once
#include "rw_kv.hpp"

namespace rw {

constexpr int SCORE_TOP = 32;         // alternatives per row at most
constexpr int SCORE_MAX_PARTS = 64;   // parts of a row: a lane each in k_score_join
constexpr int SCORE_HEADS = 8;        // alternatives up to which k_score_join compares heads
// Alternatives up to which every step's candidates are ranked at once: 1792 rows
// with 5 73 us (with 4 here, collected: 76), 366 rows with 12 28.5 (with 16 here: 33.9).
constexpr int SCORE_EAGER = 8;
constexpr int SCORE_LINE = 128;       // bytes that the loads of a step are aligned to
constexpr uint32_t SCORE_NONE = 0xFFFFFFFFu;

#if defined(__HIPCC__)

struct ScoreOut {
  const uint32_t *tokens;
  float *logprobs, *entropy;
  uint32_t *top_ids;
  float *top_lp;
  int64_t n_tok;
  int k;
};

// A part's results for k_score_join: M, S, T and its k best (rest: id NONE)
struct ScorePart {
  float m, s, t;
  int pad;
};

struct ScoreStats {
  float m, s, t;
};
// the sums of both, to the larger maximum (-inf where there is no logit; NaN sums stay)
__device__ inline ScoreStats score_join(const ScoreStats &a, const ScoreStats &b) {
  constexpr float NEG_INF = -__builtin_huge_valf();
  ScoreStats c{fmaxf(a.m, b.m), 0.0f, 0.0f};
  const float da = a.m == NEG_INF ? 0.0f : a.m - c.m, db = b.m == NEG_INF ? 0.0f : b.m - c.m;
  // a difference beyond f32's range weighs nothing (0 instead of -inf x 0)
  const float fa = __builtin_amdgcn_exp2f(da * PA_LOG2E), fb = __builtin_amdgcn_exp2f(db * PA_LOG2E);
  c.s = a.s * fa + b.s * fb;
  c.t = (a.t + fmaxf(da, -200.0f) * a.s) * fa + (b.t + fmaxf(db, -200.0f) * b.s) * fb;
  return c;
}

template <int CTRL, int ROWS = 0xf>
__device__ inline float score_dpp(float v) {
  const int i = __float_as_int(v);
  return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, ROWS, 0xf, false));
}
// the wavefront's largest value, in every lane
__device__ inline float score_wave_max(float v) {
  v = fmaxf(v, score_dpp<0x111>(v));  // row_shr 1, 2, 4, 8
  v = fmaxf(v, score_dpp<0x112>(v));
  v = fmaxf(v, score_dpp<0x114>(v));
  v = fmaxf(v, score_dpp<0x118>(v));
  v = fmaxf(v, score_dpp<0x142, 0xa>(v));  // row_bcast 15 into rows 1 and 3
  v = fmaxf(v, score_dpp<0x143, 0xc>(v));  // row_bcast 31 into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ inline float score_lane(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }

__device__ inline float score_wave_sum(float v) {
  auto add = [&](int ctrl_value) __attribute__((always_inline)) { v += __int_as_float(ctrl_value); };
  // (lanes without a source add 0)
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x111, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x112, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x114, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x118, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142, 0xa, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143, 0xc, 0xf, false));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// the lanes' sums of a wavefront
__device__ inline ScoreStats score_wave_join(const ScoreStats &st) {
  const ScoreStats a = score_join(st, ScoreStats{score_wave_max(st.m), 0.0f, 0.0f});
  return ScoreStats{a.m, score_wave_sum(a.s), score_wave_sum(a.t)};
}

template <int CTRL>
__device__ inline float score_dpp_all(float v) {  // every lane has a source
  const int i = __float_as_int(v);
  return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}
// A lower bound of the k-th largest of the wavefront's values, more than k of
// which are at least `lo` (k <= 32): the smallest of at least k groups' largest
// (groups of 64 / 2^ceil(log2 k) lanes), or of the values from lo on, moved up
// by halving while k values lie above; the k-th largest itself where that stops
// far below it (values of very unlike size, such as masks of the type's lowest).
//   Halving ends within 3 of k (286 f16 rows with 32 alternatives 30.2 us; at k
// 29.7 and one row with 5 the same, within 8 32.7), after 6 turns (after 3 36.8,
// after 10 the same).  The ranking starts 16 above k: 1792 rows that masks of the
// lowest value leave 700 logits of, 16 alternatives, 93 us, 100 without it (one such row
// 24.4 and 22.4; rows without masks the same either way).
__device__ inline float score_bound(float v, int k, float lo) {
  float w = fmaxf(v, score_dpp_all<0xB1>(v));  // pairs
  float o = score_dpp_all<0x4E>(w);            // fours
  w = k <= 16 ? fmaxf(w, o) : fminf(w, o);
  o = score_dpp_all<0x141>(w);  // mirrored within 8
  w = k <= 8 ? fmaxf(w, o) : fminf(w, o);
  o = score_dpp_all<0x140>(w);  // mirrored within 16
  w = k <= 4 ? fmaxf(w, o) : fminf(w, o);
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = score_lane(w, 16 * i);
  if (k <= 1) return fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
  float low = k <= 2 ? fminf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3])) : fminf(fminf(r[0], r[1]), fminf(r[2], r[3]));
  if (!(low >= lo)) low = -score_wave_max(v >= lo ? -v : -__builtin_huge_valf());
  float high = score_wave_max(v);
  int from = 64;
  for (int i = 0; i < 6 && from > k + 3; ++i) {
    const float mid = 0.5f * low + 0.5f * high;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(v >= mid));
    if (c >= k) low = mid, from = c;
    else high = mid;
  }
  if (from > k + 16) {
    const int lane = threadIdx.x & 63;
    int rank = 0;
#pragma unroll 8
    for (int e = 0; e < 64; ++e) {
      const float x = score_lane(v, e);
      rank += x > v || (x == v && e < lane);
    }
    const uint64_t kth = __builtin_amdgcn_ballot_w64(rank == k - 1 && v == v);
    if (kth) low = score_lane(v, __builtin_ctzll(kth));
  }
  return low;
}
// the smallest id among the lanes of `who` (at least one)
__device__ inline int score_first_id(uint64_t who, int id) {
  if (__builtin_popcountll(who) == 1) return __builtin_amdgcn_readlane(id, __builtin_ctzll(who));
  int m = who >> (threadIdx.x & 63) & 1 ? id : INT32_MAX;
  for (int s = 1; s < 64; s <<= 1) m = min(m, __shfl_xor(m, s));
  return __builtin_amdgcn_readfirstlane(m);
}
// the smallest value above x (x = +inf: NaN, which nothing reaches)
__device__ inline float score_next(float x) {
  const int b = __float_as_int(x + 0.0f);
  return x == 0.0f ? __int_as_float(1) : __int_as_float(b + (b < 0 ? -1 : 1));
}

// LDS that one wavefront's lanes write and read: its operations keep their order
__device__ inline void score_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// entry (v, i) comes before (w, j)
__device__ inline bool score_before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// The k best entries of a wavefront: lane r < n holds the r-th, the others -inf
// and NONE (which come before no entry).
struct ScoreBest {
  float v = -__builtin_huge_valf();
  int id = (int)SCORE_NONE;
  int n = 0;

  // Takes in the entries (w, i) of lanes 0 .. c - 1 (the others: -inf); sv, si:
  // k places of LDS.
  __device__ inline void take(float w, int i, int c, int k, float *sv, int *si) {
    const int lane = threadIdx.x & 63;
    if (n == k && c <= 4 + k * 3 / 8) {
      // few: each in its place, 15 instructions that wait for each other (366 rows
      // with 5 alternatives 26.4 us, none so 30.4; with 32, up to 4 so 31.9, these 30.2)
      for (int e = 0; e < c; ++e) {
        const float cv = score_lane(w, e);
        const int ci = __builtin_amdgcn_readlane(i, e);
        const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(score_before(v, id, cv, ci)));
        // the entries from `at` on move up one lane (0x138: from lane - 1)
        const float up = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x138, 0xf, 0xf, false));
        const int upi = __builtin_amdgcn_update_dpp(0, id, 0x138, 0xf, 0xf, false);
        v = lane < at ? v : lane == at ? cv : up;
        id = lane < at ? id : lane == at ? ci : upi;
        if (lane >= k) v = -__builtin_huge_valf(), id = (int)SCORE_NONE;
      }
      return;
    }
    // the old and the new ones are ranked together, eight at a time
    int rank = 0, rold = lane;
    for (int e = 0; e < n; e += 8)
#pragma unroll
      for (int j = 0; j < 8; ++j) rank += score_before(score_lane(v, e + j), __builtin_amdgcn_readlane(id, e + j), w, i);
    for (int e = 0; e < c; e += 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) rank += score_before(score_lane(w, e + j), __builtin_amdgcn_readlane(i, e + j), w, i);
      if (n)
#pragma unroll
        for (int j = 0; j < 8; ++j) rold += score_before(score_lane(w, e + j), __builtin_amdgcn_readlane(i, e + j), v, id);
    }
    score_wave_sync();
    if (lane < c && rank < k) sv[rank] = w, si[rank] = i;
    if (lane < n && rold < k) sv[rold] = v, si[rold] = id;
    score_wave_sync();
    n = min(k, n + c);
    v = lane < n ? sv[lane] : -__builtin_huge_valf();
    id = lane < n ? si[lane] : (int)SCORE_NONE;
    score_wave_sync();
  }
};

// log-probs, entropy and alternatives of a row from its sums and its k best
// (LDS; id NONE where there are fewer), by one workgroup
template <class E>
__device__ inline void score_finish(const typename E::T *x, int n, int64_t row, const ScoreStats &st, const float *bv,
                                    const int *bi, const ScoreOut &o) {
  const float nan = __builtin_nanf("");
  // NaN sums: a NaN or +inf among the logits; M = -inf: nothing else in the row
  const bool bad = !(st.s > 0.0f) || st.m == -__builtin_huge_valf();
  const float ls = logf(st.s);
  if (threadIdx.x == 0 && o.entropy) o.entropy[row] = bad ? nan : ls - st.t / st.s;
  if ((int)threadIdx.x < o.k) {
    const int id = bi[threadIdx.x];
    o.top_ids[row * o.k + threadIdx.x] = bad ? SCORE_NONE : (uint32_t)id;
    o.top_lp[row * o.k + threadIdx.x] = bad ? nan : id == (int)SCORE_NONE ? -__builtin_huge_valf() : (bv[threadIdx.x] - st.m) - ls;
  }
  for (int64_t i = threadIdx.x; i < o.n_tok; i += blockDim.x) {
    const uint32_t id = o.tokens[row * o.n_tok + i];
    float lp = nan;
    if (id == SCORE_NONE) lp = 0.0f;
    else if (id < (uint32_t)n && !bad) lp = (E::load(x + id) - st.m) - ls;
    o.logprobs[row * o.n_tok + i] = lp;
  }
}

// NJ: 16-byte loads per lane and step; NW: wavefronts.  blockIdx.x = row * parts + part.
template <class E, int NJ, int NW>
__global__ __launch_bounds__(64 * NW) void k_score(const typename E::T *__restrict__ logits, int64_t ld, int n, int parts,
                                               int64_t part_len, ScoreOut o, ScorePart *__restrict__ ps,
                                               float *__restrict__ pv, int *__restrict__ pi) {
  using T = typename E::T;
  constexpr float NEG_INF = -__builtin_huge_valf();
  constexpr int V = 16 / sizeof(T), PER = NJ * V, CAP = 64 + 64 * V;
  typedef T Vec __attribute__((ext_vector_type(V)));
  __shared__ float ev[NW][CAP + SCORE_TOP];  // per wavefront
  __shared__ int ei[NW][CAP + SCORE_TOP];
  __shared__ ScoreStats ss[NW];
  __shared__ float bv[SCORE_TOP];
  __shared__ int bi[SCORE_TOP];
  const int64_t row = blockIdx.x / parts;
  const int pt = blockIdx.x % parts, k = o.k;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T *x = logits + row * ld;
  // places count from the cache line in which the row starts
  const int skip = (int)(((uintptr_t)x & (SCORE_LINE - 1)) / sizeof(T));
  const int64_t u1 = min((int64_t)n + skip, (int64_t)(pt + 1) * part_len);

  ScoreStats st{NEG_INF, 0.0f, 0.0f};
  const float all = score_next(NEG_INF);
  float lo = all;  // the smallest logit that may be one of the k best
  ScoreBest best;
  float *wv_v = ev[wv], *sv = ev[wv] + CAP;  // candidates; the places that `take` wants
  int *wv_i = ei[wv], *si = ei[wv] + CAP;
  int cnt = 0;

  auto keep = [&]() __attribute__((always_inline)) {
    score_wave_sync();
    for (int at = 0; at < cnt; at += 64) {
      const float v = at + lane < cnt ? wv_v[at + lane] : NEG_INF;
      const int id = at + lane < cnt ? wv_i[at + lane] : INT32_MAX;
      // (of many equal logits the first ones may leave none to take in)
      if (best.n < k || __builtin_amdgcn_ballot_w64(score_before(v, id, score_lane(best.v, k - 1), __builtin_amdgcn_readlane(best.id, k - 1))))
        best.take(v, id, min(64, cnt - at), k, sv, si);
    }
    cnt = 0;
    score_wave_sync();
    if (best.n == k) lo = fmaxf(lo, score_next(score_lane(best.v, k - 1)));
  };

  // the step at place u: this lane's j-th load has the ids u - skip + (64 j + lane) V ..
  auto load = [&](int64_t u, Vec(&q)[NJ]) __attribute__((always_inline)) {
    const int64_t w0 = u - skip, e0 = w0 + lane * V;
    if (w0 >= 0 && w0 + 64 * PER <= n) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) q[j] = *(const Vec *)(x + e0 + 64 * V * j);
    } else {  // a step that the row does not fill
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int64_t e = e0 + 64 * V * j + i;
          q[j][i] = e >= 0 && e < n ? x[e] : (T)NEG_INF;
        }
    }
  };
  Vec ahead[NJ];  // the next step, on its way while this one is worked on
  int64_t u = (int64_t)pt * part_len + wv * 64 * PER;
  if (u < u1) load(u, ahead);
  for (; u < u1; u += 64 * NW * PER) {
    const int64_t e0 = u - skip + lane * V;
    float y[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) y[j] = (float)ahead[j / V][j % V];
    if (u + 64 * NW * PER < u1) load(u + 64 * NW * PER, ahead);
    float mx = y[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) mx = fmaxf(mx, y[j]);
    {
      const ScoreStats none{mx, 0.0f, 0.0f};
      if (mx > st.m) st = score_join(st, none);
      const float m0 = st.m == NEG_INF ? 0.0f : st.m;
      float s = 0.0f, t = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float d = y[j] - m0, e = __builtin_amdgcn_exp2f(d * PA_LOG2E);
        s += e;
        t = fmaf(fmaxf(d, -200.0f), e, t);
      }
      st.s += s, st.t += t;
    }
    if (k == 0) continue;
    const uint64_t pass = __builtin_amdgcn_ballot_w64(mx >= lo);
    if (!pass) continue;
    // the k-th largest of the lanes' maxima so far is one of the k best (looked for
    // where more than 4 lanes pass: 1792 rows with 16 alternatives 78.8 us, with 32
    // 101; more than 1: 80.4, 108; more than 12: 81.5, 96; up to 8 alternatives
    // k + 3 lanes, k or k + 12 the same)
    if (__builtin_popcountll(pass) > (k <= SCORE_EAGER ? k + 3 : 4) && __builtin_popcountll(__builtin_amdgcn_ballot_w64(st.m >= all)) > k)
      lo = fmaxf(lo, score_bound(st.m, k, all));
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float mj = y[j * V];
#pragma unroll
      for (int i = 1; i < V; ++i) mj = fmaxf(mj, y[j * V + i]);
      if (!__builtin_amdgcn_ballot_w64(mj >= lo)) continue;
      if (cnt > CAP - 64 * V) keep();  // equal logits in great number
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint64_t in = __builtin_amdgcn_ballot_w64(y[j * V + i] >= lo);
        if (!in) continue;
        if (y[j * V + i] >= lo) {
          const int at = cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
          wv_v[at] = y[j * V + i], wv_i[at] = (int)(e0 + 64 * V * j + i);
        }
        cnt += __builtin_popcountll(in);
      }
    }
    if (cnt && (k <= SCORE_EAGER || cnt + best.n > 64)) keep();
  }
  if (cnt) keep();

  // lanes, then wavefronts
  st = score_wave_join(st);
  if (NW == 1) {
    if (lane < SCORE_TOP) bv[lane] = best.v, bi[lane] = best.id;
    score_wave_sync();
  } else {
    if (threadIdx.x < SCORE_TOP) bv[threadIdx.x] = NEG_INF, bi[threadIdx.x] = (int)SCORE_NONE;
    if (lane == 0) ss[wv] = st;
    if (lane < SCORE_TOP) ev[wv][lane] = best.v, ei[wv][lane] = best.id;
    __syncthreads();
    st = score_join(ss[0], ss[NW - 1]);
#pragma unroll
    for (int c = 1; c < NW - 1; ++c) st = score_join(st, ss[c]);
    if (lane < k) {
      int rank = lane;
#pragma unroll
      for (int c = 0; c < NW; ++c)
        if (c != wv)
#pragma unroll 8
          for (int e = 0; e < k; ++e) rank += score_before(ev[c][e], ei[c][e], best.v, best.id);
      if (lane < best.n && rank < k) bv[rank] = best.v, bi[rank] = best.id;
    }
    __syncthreads();
  }
  if (parts == 1) {
    score_finish<E>(x, n, row, st, bv, bi, o);
  } else {
    if (threadIdx.x == 0) ps[blockIdx.x] = ScorePart{st.m, st.s, st.t, 0};
    if ((int)threadIdx.x < k) {
      pv[(int64_t)blockIdx.x * k + threadIdx.x] = bv[threadIdx.x];
      pi[(int64_t)blockIdx.x * k + threadIdx.x] = bi[threadIdx.x];
    }
  }
}

// The parts of a row: sums in order, and the k best of the parts' lists.
// K = 1 (few alternatives): the best of the lists' heads, a lane a list, k
// times.  Else by halving the number of lists: of two lists of K places, one
// read backwards, the better entry of each place is one of the K best, and
// log2 K exchanges put these in order again, 64 / K pairs of lists per
// wavefront and turn.  (51 lists of 5: 3.5 us against 5.0; of 16: 6.3 and 6.4;
// of 32: 11.0 and 9.9; 341 rows of 6 lists of 10: 5.1 and 4.2.)
template <class E, int K>
__global__ __launch_bounds__(256) void k_score_join(const typename E::T *__restrict__ logits, int64_t ld, int n, int parts,
                                                    ScoreOut o, const ScorePart *__restrict__ ps,
                                                    const float *__restrict__ pv, const int *__restrict__ pi) {
  constexpr float NEG_INF = -__builtin_huge_valf();
  constexpr int LIST = K == 1 ? SCORE_HEADS : K;
  __shared__ float lv[SCORE_MAX_PARTS * LIST], bv[SCORE_HEADS];
  __shared__ int li[SCORE_MAX_PARTS * LIST], bi[SCORE_HEADS];
  const int64_t row = blockIdx.x;
  const int k = o.k, lane = threadIdx.x & 63;
  for (int e = threadIdx.x; e < parts * LIST; e += 256) {
    const int p = e / LIST, r = e % LIST;
    const bool in = r < k;
    lv[e] = in ? pv[(row * parts + p) * k + r] : NEG_INF;
    li[e] = in ? pi[(row * parts + p) * k + r] : (int)SCORE_NONE;
  }
  ScoreStats st{NEG_INF, 0.0f, 0.0f};
  if (lane < parts) {
    const ScorePart p = ps[row * parts + lane];
    st = ScoreStats{p.m, p.s, p.t};
  }
  st = score_wave_join(st);
  __syncthreads();
  if (K == 1) {
    if (threadIdx.x < 64 && k) {
      int at = 0;
      float v = lane < parts ? lv[lane * LIST] : NEG_INF;
      int id = lane < parts ? li[lane * LIST] : (int)SCORE_NONE;
      for (int r = 0; r < k; ++r) {
        // (where no entry is left, all heads are -inf and NONE: one of them is written)
        const float top = score_wave_max(v);
        const int first = score_first_id(__builtin_amdgcn_ballot_w64(v == top), id);
        if (lane == __builtin_ctzll(__builtin_amdgcn_ballot_w64(v == top && id == first))) {
          bv[r] = v, bi[r] = id;
          ++at;
          v = lane < parts && at < k ? lv[lane * LIST + at] : NEG_INF;
          id = lane < parts && at < k ? li[lane * LIST + at] : (int)SCORE_NONE;
        }
      }
    }
    __syncthreads();
    score_finish<E>(logits + row * ld, n, row, st, bv, bi, o);
    return;
  }
  // lists p and p + half become list p
  for (int lists = parts; lists > 1; lists = (lists + 1) / 2) {
    const int half = (lists + 1) / 2;
    for (int p0 = 0; p0 < half; p0 += 256 / K) {
      const int p = p0 + threadIdx.x / K, r = threadIdx.x % K;
      float v = NEG_INF;
      int id = (int)SCORE_NONE;
      if (p + half < lists) {
        v = lv[p * K + r], id = li[p * K + r];
        const float w = lv[(p + half) * K + K - 1 - r];
        const int i = li[(p + half) * K + K - 1 - r];
        if (score_before(w, i, v, id)) v = w, id = i;
#pragma unroll
        for (int x = K / 2; x; x >>= 1) {
          // the lower lane of a pair keeps the better one (lanes of one list take this branch together)
          const float y = __shfl_xor(v, x);
          const int j = __shfl_xor(id, x);
          if (score_before(y, j, v, id) == !(r & x) && (y != v || j != id)) v = y, id = j;
        }
        lv[p * K + r] = v, li[p * K + r] = id;
      }
    }
    __syncthreads();
  }
  score_finish<E>(logits + row * ld, n, row, st, lv, li, o);
}

#endif  // __HIPCC__

}  // namespace rw
