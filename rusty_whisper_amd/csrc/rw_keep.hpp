// rw_keep.hpp -- which drafted tokens are accepted, and their rows moved together.
#pragma once
#include "rw_kv8.hpp"

namespace rw {

#if defined(__HIPCC__)

// Rows past + kept[j] of a tree's sequence become its rows past + j, every layer.  kept
// rises, so kept[j] >= j and no row is written before it was read: a row j is the
// source of no later one.  Sources are read KEEP at a time, then written; an
// entry that does not rise above its place (kept[j] <= j) moves nothing.
//   blockIdx.x: tree, y: layer, z: 2 x pieces of 256 threads of k (even) or v.  A thread
// moves 16 bytes of k's rows, or one value of v's, whose rows are innermost, so that every value
// lies in a line of its own.
//   Bound by those lines: 48 trees of 3 rows to move, 24 layers of 8 heads of 128, f16: 1.2
// million of them read and written, 41 us, for 28 MB that move (four layers per workgroup: 48).
constexpr int KEEP = 4;
template <class T>
__global__ __launch_bounds__(256) void k_kv_keep(PagedView w, int64_t layer_rows, const int32_t *__restrict__ past,
                                                 const int32_t *__restrict__ kept, int64_t ld_kept,
                                                 const int32_t *__restrict__ count, int most) {
  constexpr int V = 16 / sizeof(T);
  __shared__ int64_t base[KEEP][2];  // where the page of a source and of its destination begins, in rows; -1: no move
  __shared__ int slot[KEEP][2];
  const int tree = blockIdx.x, t = threadIdx.x;
  const int n = min(count[tree], most), p0 = past[tree];
  const bool is_v = blockIdx.z & 1;
  const int i = (blockIdx.z >> 1) * 256 + t, all = w.heads * w.dim;
  const int64_t layer = blockIdx.y * layer_rows;  // rows (of one head) before this layer
  T *k = (T *)w.k + layer * w.dim, *v = (T *)w.v + layer * w.dim;
  const int kh = i * V / w.dim, kd = i * V % w.dim;
  for (int j0 = 0; j0 < n; j0 += KEEP) {
    __syncthreads();
    if (t < KEEP) {
      const int j = j0 + t, from = j < n ? kept[tree * ld_kept + j] : j;
      int a = -1, b = -1, sa = 0, sb = 0;
      if (from > j && p0 >= 0 && from <= INT32_MAX - p0)
        a = kv_place(w, tree, p0 + from, &sa), b = kv_place(w, tree, p0 + j, &sb);
      const bool move = a >= 0 && b >= 0;
      base[t][0] = move ? (int64_t)a * w.heads << w.pr : -1, slot[t][0] = sa;
      base[t][1] = move ? (int64_t)b * w.heads << w.pr : -1, slot[t][1] = sb;
    }
    __syncthreads();
    // element e of the row j's side s: 16 bytes of k, a value of v, a scale
    auto at_k = [&](int j, int s) { return (u32x4 *)(k + (base[j][s] + ((int64_t)kh << w.pr) + slot[j][s]) * w.dim + kd); };
    auto at_v = [&](int j, int s) { return v + base[j][s] * w.dim + ((int64_t)i << w.pr) + slot[j][s]; };
    auto at_s = [&](int j, int s) { return (is_v ? w.vs : w.ks) + layer + base[j][s] + ((int64_t)i << w.pr) + slot[j][s]; };
#define RW_MOVE(TYPE, AT)                                          \
  do {                                                             \
    TYPE x[KEEP] = {};                                             \
    _Pragma("unroll") for (int j = 0; j < KEEP; ++j)               \
      if (base[j][0] >= 0) x[j] = *AT(j, 0);                       \
    _Pragma("unroll") for (int j = 0; j < KEEP; ++j)               \
      if (base[j][0] >= 0) *AT(j, 1) = x[j];                       \
  } while (0)
    if (!is_v && i < all / V) RW_MOVE(u32x4, at_k);
    if (is_v && i < all) RW_MOVE(T, at_v);
    if (w.ks && i < w.heads) RW_MOVE(float, at_s);
#undef RW_MOVE
  }
}

// The path of a tree that its samples agree with: from the root (node 0, always
// kept) to the first child that holds the sample of its parent, and on.  A child
// comes behind its parent, so the walk ends.  One wavefront per tree; trees
// up to ACCEPT nodes are walked in LDS, where a step takes no trip to memory (48 trees of 48: 4.9 us; one of 13: 2.2).
constexpr int ACCEPT = 1024;
__global__ __launch_bounds__(64) void k_tree_accept(const uint32_t *__restrict__ tokens, const int32_t *__restrict__ parent,
                                                    const uint32_t *__restrict__ sampled, int rows,
                                                    const int32_t *__restrict__ starts, int most,
                                                    int32_t *__restrict__ kept, int64_t ld_kept,
                                                    int32_t *__restrict__ count, uint32_t *__restrict__ next) {
  __shared__ uint32_t st[ACCEPT], ss[ACCEPT];
  __shared__ int sp[ACCEPT];
  const int tree = blockIdx.x, lane = threadIdx.x;
  // (an end below zero is taken as zero: its distance from s0 could pass 32 bits and come out positive)
  const int s0 = starts[tree], n = s0 < 0 ? 0 : min(min(max(starts[tree + 1], 0), rows) - s0, most);
  const uint32_t *tok = tokens + s0, *smp = sampled + s0;
  const int32_t *par = parent + s0;
  if (n > 0 && n <= ACCEPT) {
    for (int j = lane; j < n; j += 64) st[j] = tok[j], ss[j] = smp[j], sp[j] = par[j];
    __syncthreads();
    tok = st, smp = ss, par = sp;
  }
  int32_t *out = kept + tree * ld_kept;
  int c = 0;
  uint32_t want = 0xFFFFFFFFu;
  for (int at = 0; at >= 0 && at < n;) {
    if (lane == 0) out[c] = at;
    ++c;
    want = smp[at];
    int found = -1;
    for (int j0 = at + 1; j0 < n && found < 0; j0 += 64) {
      const int j = j0 + lane;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(j < n && par[min(j, n - 1)] == at && tok[min(j, n - 1)] == want);
      if (hit) found = j0 + __builtin_ctzll(hit);
    }
    at = found;
  }
  for (int j = c + lane; j < most; j += 64) out[j] = -1;
  if (lane == 0) count[tree] = c, next[tree] = want;
}

#endif  // __HIPCC__

}  // namespace rw
