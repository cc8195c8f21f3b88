// rw_draft.hip -- the entries of include/rw_rocm.h for programs that draft
// tokens: attention of several new rows per sequence (trees, chunks of
// prompts, single rows over 8-bit pages), sampling, and what becomes of the accepted path.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "rw_keep.hpp"
#include "rw_rocm.h"
#include "rw_sample.hpp"
#include "rw_serve.hpp"
#include "rw_tree.hpp"

using namespace rw;

// ------------------------------------------------------------ attention

namespace rw {

// How a launch cuts its trees' queries and keys, as PagedPlan does for single rows.
// Queries: 16 per workgroup where no more are there, and for f32, for which k_tree_shared has no
// form.  64 with keys and values through LDS otherwise; f16 pools 128 from 65 on, since each value is
// there in two parts and a part read from LDS then has two products: 4 chunks of 512 rows behind 4100, 8
// heads of 4 x 128: 466 us by 128, 538 by 64; bf16 557 and 439, int8 636 and 471, e4m3 514 and 447.  (f32 by 16:
// 1980 us, where the products alone take 955 at a large f32 product's rate; by more is not built.)
// Keys: in one chunk up to 256 KB a head.  One tree is cut as far as the join goes, a batch
// into chunks of 192 KB, but no more workgroups in all than fill the device's 512 places four times over,
// the cap that acts in large batches.  By caps: 61 single rows of up to 8191 keys, 8 heads of 4 x 128, e4m3: 600
// 121 us, 1024 (2 chunks) 112, 2048 (4, of 528 KB) 106, 4096 (8) 112, 8192 (11) 116; 24 trees of up to 48 rows, up to
// 6048 keys, int8: 1024 (1) 272, 1200 (2) 178, 2048 (3) 188, 4096 (7) 172, 8192 (9) 176.  By sizes, where the cap leaves
// the choice: 8 such rows by 96 KB 38 us, 192 30, 384 29; 4 such trees 65, 68, 78.
struct TreePlan {
  int nq;         // queries per workgroup: 16 (k_tree_attn), 64 or 128 (k_tree_shared)
  size_t qtiles;  // workgroups per tree, key head and chunk
  int chunk, nsplit;
  size_t most;
};
static TreePlan tree_plan(const rw_kv_pages *p, int n_head, size_t n_trees, size_t max_rows, size_t max_len) {
  TreePlan L{};
  const size_t queries = (size_t)n_head / p->n_head * max_rows;
  max_len = std::min(max_len, (size_t)1 << 30);
  L.nq = queries <= 16 || p->dtype == RW_F32 ? 16 : p->dtype == RW_F16 && queries > 64 ? 128 : 64;
  L.qtiles = cdiv(queries, L.nq);
  const size_t base = n_trees * p->n_head * L.qtiles;
  const size_t bytes = max_len * 2 * (p->head_size * pool_size(p->dtype) + (scaled(p->dtype) ? 4 : 0));
  size_t nsplit = 1;
  if (bytes > (size_t)256 << 10) {
    nsplit = std::min(cdiv(bytes, (size_t)128 << 10), (size_t)PA_MAX_SPLIT / base);
    if (n_trees > 1)
      nsplit = std::max(nsplit, std::min(cdiv(bytes, (size_t)192 << 10), std::min((size_t)2048, 256 * n_trees) / base));
    nsplit = std::max((size_t)1, nsplit);
  }
  L.most = nsplit;
  L.chunk = (int)(cdiv(std::max(max_len, (size_t)1), nsplit * 128) * 128);
  L.nsplit = (int)std::max((size_t)1, cdiv(max_len, (size_t)L.chunk));
  return L;
}

size_t tree_workspace(const rw_kv_pages *p, int n_head, size_t rows, size_t n_trees, size_t max_rows, size_t max_len) {
  const TreePlan L = tree_plan(p, n_head, n_trees, max_rows, max_len);
  return L.most > 1 ? rows * n_head * L.most * (p->head_size + 2) * 4 : 0;
}

template <class E, int DH>
static int launch_tree(const TreeArgs &a, const TreePlan &L, size_t join, hipStream_t s) {
  const dim3 grid((unsigned)(cdiv((size_t)a.n_trees * a.kv_heads, 8) * 8 * L.qtiles), (unsigned)L.nsplit);
  auto *kernel = k_tree_attn<E, DH>;
  if constexpr (!std::is_same_v<E, F32>)
    if (L.nq > 16)
      kernel = 1 << a.pr >= TreeShared<E, DH>::KEYS ? k_tree_shared<E, DH, 1, true> : k_tree_shared<E, DH, 1, false>;
  if constexpr (std::is_same_v<E, F16>)
    if (L.nq > 64)
      kernel = 1 << a.pr >= TreeShared<E, DH>::KEYS ? k_tree_shared<E, DH, 2, true> : k_tree_shared<E, DH, 2, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a);
  SERVE_TRY(launched(L.nq > 16 ? "k_tree_shared" : "k_tree_attn"));
  if (L.nsplit == 1) return RW_OK;
  if (L.nsplit <= JOIN_FEW)
    hipLaunchKernelGGL((k_tree_join_few<DH>), dim3((unsigned)cdiv(join, 4)), dim3(256), 0, s, a, L.nsplit, L.nq, (int)join);
  else
    hipLaunchKernelGGL((k_tree_join<DH>), dim3((unsigned)join), dim3(256), 0, s, a, L.nsplit, L.nq);
  return launched("k_tree_join");
}

template <class E>
static int launch_tree_dim(int dim, const TreeArgs &a, const TreePlan &L, size_t join, hipStream_t s) {
  switch (dim) {
    case 32: return launch_tree<E, 32>(a, L, join, s);
    case 64: return launch_tree<E, 64>(a, L, join, s);
    case 96: return launch_tree<E, 96>(a, L, join, s);
    default: return launch_tree<E, 128>(a, L, join, s);
  }
}

int tree_launch(const TreeCall &c, const rw_kv_pages *p, void *ws, hipStream_t s) {
  const PagedView &w = c.w;
  const size_t max_len = std::min(c.max_len, std::min((size_t)1 << 30, (size_t)w.ld << w.pr));
  const TreePlan L = tree_plan(p, c.n_head, c.n_trees, c.max_rows, max_len);
  TreeArgs a{};
  a.k = w.k, a.v = w.v, a.ks = w.ks, a.vs = w.vs;
  a.q = c.q, a.ldq = c.ldq, a.out = c.out, a.ldo = c.ldo, a.part = (float *)ws;
  a.table = w.table, a.seq = w.seq, a.ld_table = w.ld, a.starts = c.starts, a.past = c.past;
  a.mask = c.mask, a.n_words = c.n_words;
  a.rows = (int)c.rows, a.n_trees = (int)c.n_trees, a.max_rows = (int)c.max_rows, a.kv_heads = w.heads;
  a.group = c.n_head / w.heads, a.pr = w.pr, a.n_pages = w.n_pages, a.n_seqs = w.n_seqs;
  a.max_len = (int)max_len, a.chunk = L.chunk, a.qtiles = (int)L.qtiles;
  const size_t join = c.n_trees * c.max_rows * c.n_head;
  switch (c.dtype) {
    case RW_F32: return launch_tree_dim<F32>(w.dim, a, L, join, s);
    case RW_F16: return launch_tree_dim<F16>(w.dim, a, L, join, s);
    case RW_BF16: return launch_tree_dim<BF16>(w.dim, a, L, join, s);
    case RW_I8: return launch_tree_dim<I8>(w.dim, a, L, join, s);
    default: return launch_tree_dim<E4M3>(w.dim, a, L, join, s);
  }
}

}  // namespace rw

// trees of a call: each at most max_rows rows
static int check_trees(size_t n_trees, size_t max_rows, int n_head) {
  if (n_trees > MOST_ROWS || max_rows > MOST_ROWS) return fail(RW_EINVAL, "%zu trees of up to %zu rows", n_trees, max_rows);
  if (n_trees * max_rows > MOST_ROWS / n_head)
    return fail(RW_EINVAL, "%zu trees of up to %zu rows of %d heads", n_trees, max_rows, n_head);
  return RW_OK;
}

// -------------------------------------------------------------- entries

extern "C" {

size_t rw_rocm_tree_attention_workspace_size(const rw_kv_pages *pages, size_t rows, int n_head, size_t n_trees,
                                             size_t max_rows, size_t max_len) {
  if (check_pages(pages) || check_paged_heads(pages, rows, n_head, max_len) || check_trees(n_trees, max_rows, n_head)) return 0;
  if (rows == 0 || n_trees == 0 || max_rows == 0) return 0;
  return tree_workspace(pages, n_head, rows, n_trees, max_rows, max_len);
}

int rw_rocm_tree_attention_dev(const rw_kv_pages *pages, size_t layer, const float *q, size_t ldq, size_t rows, int n_head,
                               const int32_t *table, size_t ld_table, size_t n_seqs, const int32_t *seq, size_t n_trees,
                               const int32_t *starts, size_t max_rows, const int32_t *past, const uint32_t *mask,
                               size_t n_words, size_t max_len, float *out, size_t ldo, void *workspace,
                               size_t workspace_len, void *stream) {
  SERVE_TRY(check_pages(pages));
  if (layer >= pages->n_layer) return fail(RW_EINVAL, "layer %zu of %zu", layer, pages->n_layer);
  SERVE_TRY(check_paged_heads(pages, rows, n_head, max_len));
  SERVE_TRY(check_trees(n_trees, max_rows, n_head));
  if (rows == 0 || n_trees == 0 || max_rows == 0) return RW_OK;
  const size_t n = (size_t)n_head * pages->head_size;
  SERVE_TRY(check_rows(q, ldq, n, "q"));
  SERVE_TRY(check_rows(out, ldo, n, "out"));
  SERVE_TRY(check_table(table, ld_table, n_seqs, n_trees, seq, past, "past"));
  if (!starts || !aligned(starts, 4)) return fail(RW_EINVAL, "starts is NULL or not 4-byte aligned");
  if (mask && (!aligned(mask, 4) || n_words < 1 || n_words > MOST_ROWS))
    return fail(RW_EINVAL, "a mask of %zu words per row, 4-byte aligned", n_words);
  int dev;
  SERVE_TRY(call_device(pages->k, "the pages' k", &dev));
  CallWorkspace hold;
  void *ws = nullptr;
  SERVE_TRY(hold.take(dev, workspace, workspace_len, tree_workspace(pages, n_head, rows, n_trees, max_rows, max_len), stream, &ws));
  return tree_launch(TreeCall{paged_view(pages, layer, table, ld_table, n_seqs, seq), pages->dtype, q, (int64_t)ldq, rows, n_head,
                              n_trees, starts, past, max_rows, mask, (int)n_words, max_len, out, (int64_t)ldo},
                     pages, ws, (hipStream_t)stream);
}

int rw_rocm_tree_accept_dev(const uint32_t *tokens, const int32_t *parent, const uint32_t *sampled, size_t rows,
                            const int32_t *starts, size_t n_trees, size_t max_rows, int32_t *kept, int32_t *n_kept,
                            uint32_t *next, void *stream) {
  if (rows > MOST_ROWS) return fail(RW_EINVAL, "rows = %zu: at most %zu", rows, MOST_ROWS);
  SERVE_TRY(check_trees(n_trees, max_rows, 1));
  if (n_trees == 0) return RW_OK;
  if (!starts || !n_kept || !next || (max_rows && !kept)) return fail(RW_EINVAL, "starts, kept, n_kept or next is NULL");
  if (rows && max_rows && (!tokens || !parent || !sampled)) return fail(RW_EINVAL, "tokens, parent or sampled is NULL");
  if (!aligned(tokens, 4) || !aligned(parent, 4) || !aligned(sampled, 4) || !aligned(starts, 4) || !aligned(kept, 4) ||
      !aligned(n_kept, 4) || !aligned(next, 4))
    return fail(RW_EINVAL, "the arrays must be 4-byte aligned");
  int dev;
  SERVE_TRY(call_device(starts, "starts", &dev));
  hipLaunchKernelGGL(k_tree_accept, dim3((unsigned)n_trees), dim3(64), 0, (hipStream_t)stream, tokens, parent, sampled,
                     (int)rows, starts, (int)max_rows, kept, (int64_t)max_rows, n_kept, next);
  return launched("k_tree_accept");
}

int rw_rocm_kv_keep_rows_dev(const rw_kv_pages *pages, const int32_t *table, size_t ld_table, size_t n_seqs,
                             const int32_t *seq, size_t n_trees, const int32_t *past, const int32_t *kept, size_t ld_kept,
                             const int32_t *n_kept, void *stream) {
  SERVE_TRY(check_pages(pages));
  SERVE_TRY(check_trees(n_trees, 1, 1));
  if (n_trees == 0 || ld_kept == 0) return RW_OK;
  SERVE_TRY(check_table(table, ld_table, n_seqs, n_trees, seq, past, "past"));
  if (ld_kept > MOST_ROWS) return fail(RW_EINVAL, "%zu rows kept per tree: at most %zu", ld_kept, MOST_ROWS);
  if (!kept || !n_kept || !aligned(kept, 4) || !aligned(n_kept, 4)) return fail(RW_EINVAL, "kept or n_kept is NULL or not 4-byte aligned");
  int dev;
  SERVE_TRY(call_device(pages->k, "the pages' k", &dev));
  const size_t n = (size_t)pages->n_head * pages->head_size;
  const int64_t layer = (int64_t)pages->n_pages * pages->n_head * pages->page_rows;
  // (a launch has fewer than 2^32 threads: layers and trees in as many launches as that takes)
  const dim3 block(256);
  const size_t z = 2 * cdiv(n, 256), layers = std::min((size_t)pages->n_layer, std::max((size_t)1, MOST_ROWS / z));
  const size_t trees = std::max((size_t)1, MOST_ROWS / (z * layers));
  for (size_t l0 = 0; l0 < pages->n_layer; l0 += layers)
    for (size_t t0 = 0; t0 < n_trees; t0 += trees) {
      PagedView u = paged_view(pages, l0, table, ld_table, n_seqs, seq);
      if (seq) u.seq = seq + t0;
      else u.table = table + t0 * ld_table, u.n_seqs = (int)(n_seqs - t0);
      const dim3 grid((unsigned)std::min(trees, n_trees - t0), (unsigned)std::min(layers, pages->n_layer - l0), (unsigned)z);
#define RW_KEEP(T)                                                                                                     \
  hipLaunchKernelGGL((k_kv_keep<T>), grid, block, 0, (hipStream_t)stream, u, layer, past + t0, kept + t0 * ld_kept, \
                     (int64_t)ld_kept, n_kept + t0, (int)ld_kept)
      if (pool_size(pages->dtype) == 4) RW_KEEP(uint32_t);
      else if (pool_size(pages->dtype) == 2) RW_KEEP(uint16_t);
      else RW_KEEP(uint8_t);
#undef RW_KEEP
      SERVE_TRY(launched("k_kv_keep"));
    }
  return RW_OK;
}

// (a row's histograms are in its workgroup's LDS)
size_t rw_rocm_sample_tokens_workspace_size(size_t, size_t) { return 0; }

int rw_rocm_sample_tokens_dev(int dtype, const void *logits, size_t ld, size_t rows, size_t n_vocab, const float *u,
                              const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                              uint32_t *tokens, float *logprobs, void *workspace, size_t workspace_len, void *stream) {
  if (!elem_size(dtype)) return fail(RW_EINVAL, "unsupported dtype %d (RW_F32, RW_F16 or RW_BF16)", dtype);
  if (n_vocab < 1 || n_vocab > SAMPLE_VOCAB) return fail(RW_EINVAL, "n_vocab = %zu: between 1 and %zu", n_vocab, SAMPLE_VOCAB);
  if (rows > MOST_ROWS) return fail(RW_EINVAL, "rows = %zu: at most %zu", rows, MOST_ROWS);
  if (rows == 0) return RW_OK;
  if (!logits || !aligned(logits, elem_size(dtype))) return fail(RW_EINVAL, "logits is NULL or not aligned");
  if (ld < n_vocab || ld > ((size_t)1 << 40)) return fail(RW_EINVAL, "logits: row stride %zu for rows of %zu", ld, n_vocab);
  if (!u || !tokens) return fail(RW_EINVAL, "u or tokens is NULL");
  if (!aligned(u, 4) || !aligned(temperature, 4) || !aligned(top_k, 4) || !aligned(top_p, 4) || !aligned(min_p, 4) ||
      !aligned(tokens, 4) || !aligned(logprobs, 4))
    return fail(RW_EINVAL, "settings and results must be 4-byte aligned");
  int dev;
  SERVE_TRY(call_device(logits, "logits", &dev));
  CallWorkspace hold;
  void *ws = nullptr;
  SERVE_TRY(hold.take(dev, workspace, workspace_len, rw_rocm_sample_tokens_workspace_size(rows, n_vocab), stream, &ws));
  const SampleArgs a{u, temperature, top_k, top_p, min_p, tokens, logprobs, (int64_t)ld, (int)n_vocab, (int)rows};
  return sample_launch(dtype, logits, a, rows, (hipStream_t)stream);
}

}  // extern "C"
