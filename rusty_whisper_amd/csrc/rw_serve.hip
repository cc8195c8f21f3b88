// rw_serve.hip -- the entries of include/rw_rocm.h for programs that serve
// many sequences: keys and values in pages (writes, copies, attention, the
// book of pages) and the scoring of tokens.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <stdexcept>
#include <vector>

#include "rw_kv.hpp"
#include "rw_kv8.hpp"
#include "rw_kvbook.hpp"
#include "rw_rocm.h"
#include "rw_score.hpp"
#include "rw_serve.hpp"

using namespace rw;

// ------------------------------------------------------------ attention

// How a launch cuts its rows' keys: chunks of `chunk` keys, `nsplit` of them
// for the longest row.  `most`, of which the workspace's size is made, is no
// less than nsplit and never falls with max_len.
//   Up to 256 KB of k and v per row and head: one chunk.  A CU draws 50 GB/s,
// so 256 KB take it 5 us, and the join's launch takes 3 to 5 (448 f16 keys of
// 64, 5 rows: 6.5 us, in two chunks 8.4; 1024 keys of 128, 512 KB: 14.9 against
// 9.9 in four).
//   Longer: chunks of 128 KB or more, up to 512 workgroups, two per CU (more of
// them only cost: 131071 keys over 8 heads in 512 workgroups 99 us, in 1024 102,
// in 2048 110).
//   Several rows are seldom of one length, and a long one must not be left to
// itself at the end: up to 256 workgroups per row and 4096 in all, in chunks of
// 192 KB or more (48 ragged f32 rows of 20 heads: 58.2 us; chunks of 256 KB 61.2,
// of 384 KB 68.5, of 128 KB 58.4; 11 rows of 10468 keys, 8 heads: 88.5 to 89 with
// any; four f16 rows of 32768 keys, 8 heads: 97 us, ragged 72, and with up to 4096
// 102 and 79).  Equal shares of all rows' keys for 512 resident workgroups, found from
// the lengths on the device, measured 171 us where this took 157 (61 ragged
// rows, 8 heads).
struct PagedPlan {
  size_t base;  // workgroups per chunk
  int chunk, nsplit;
  size_t most;
  size_t runs;  // partial results
};
static PagedPlan paged_plan(const rw_kv_pages *p, size_t rows, int n_head, size_t max_len) {
  PagedPlan L{};
  const size_t group = (size_t)n_head / p->n_head;
  max_len = std::min(max_len, (size_t)1 << 30);
  L.base = rows * p->n_head * cdiv(group, 16);
  const size_t bytes = max_len * 2 * p->head_size * pool_size(p->dtype);
  size_t nsplit = 1;
  if (bytes > (size_t)256 << 10) {
    nsplit = std::min(cdiv(bytes, (size_t)128 << 10), (size_t)PA_MAX_SPLIT / L.base);
    if (rows > 1)
      nsplit = std::max(nsplit, std::min(cdiv(bytes, (size_t)192 << 10), std::min((size_t)4096, 256 * rows) / L.base));
    nsplit = std::max((size_t)1, nsplit);  // <= PA_MAX_SPLIT: base is no less than rows
  }
  L.most = nsplit;
  L.chunk = (int)(cdiv(std::max(max_len, (size_t)1), nsplit * 128) * 128);
  L.nsplit = (int)std::max((size_t)1, cdiv(max_len, (size_t)L.chunk));
  L.runs = rows * n_head * (size_t)L.nsplit;
  return L;
}
static size_t paged_bytes(const PagedPlan &L, size_t rows, int n_head, int head_size) {
  return L.most > 1 ? rows * n_head * L.most * (head_size + 2) * 4 : 0;
}

struct PagedCall {
  PagedView w;
  const float *q;
  int64_t ldq;
  int rows, n_head, max_len;
  const int32_t *len;
  float *out;
  int64_t ldo;
  float *part;
};

template <class E, int DH>
static int launch_paged(const PagedCall &c, const PagedPlan &L, hipStream_t s) {
  const PagedView &w = c.w;
  const int group = c.n_head / w.heads;
  const size_t items = (size_t)c.rows * w.heads;
  const dim3 grid((unsigned)(cdiv(items, 8) * 8 * cdiv(group, 16)), (unsigned)L.nsplit);
  auto *kernel = k_paged_attn<E, DH, false>;
  if constexpr (std::is_same_v<E, F16>)
    if (group == 1) kernel = k_paged_attn<E, DH, true>;
  hipLaunchKernelGGL(kernel, grid, dim3(64 * PA_WAVES), 0, s, w.k, w.v, c.q, w.table, w.seq, c.len, c.out, c.part,
                     c.rows, w.heads, group, w.pr, w.n_pages, w.n_seqs, w.ld, c.ldq, c.ldo, c.max_len, L.chunk);
  SERVE_TRY(launched("k_paged_attn"));
  if (L.nsplit == 1) return RW_OK;
  hipLaunchKernelGGL((k_paged_join<DH>), dim3((unsigned)(c.rows * c.n_head)), dim3(256), 0, s, c.part, w.seq, c.len,
                     w.n_seqs, w.ld << w.pr, c.max_len, L.chunk, L.nsplit, c.n_head, (int64_t)L.runs, c.out, c.ldo);
  return launched("k_paged_join");
}

template <class E>
static int launch_paged_dim(const PagedCall &c, const PagedPlan &L, hipStream_t s) {
  switch (c.w.dim) {
    case 32: return launch_paged<E, 32>(c, L, s);
    case 64: return launch_paged<E, 64>(c, L, s);
    case 96: return launch_paged<E, 96>(c, L, s);
    default: return launch_paged<E, 128>(c, L, s);
  }
}

// ------------------------------------------------------------- scores

// Parts of a row of logits, one workgroup each: about 2048 workgroups where rows
// are few, no part below 1024 logits.  Short parts take one wavefront, which has
// no lists to join with another's (one row of 51866, 5 alternatives: 4.4 us and
// 3.8 for the join; 26 parts of four wavefronts 6.5 and 3.6, one workgroup of
// 16 wavefronts 25).  Long ones take two (1792 rows with 5 alternatives 71 us,
// with four wavefronts, each with k best of its own, 80).
struct ScorePlan {
  int parts;
  int64_t part_len;
  bool wide;  // two wavefronts per part, else one
  size_t off_v, off_i, bytes;
};
static ScorePlan score_plan(size_t rows, size_t n_vocab, size_t k) {
  ScorePlan L{};
  const size_t places = n_vocab + SCORE_LINE / 2 - 1;  // a row may begin anywhere in its first cache line
  const size_t parts = std::max((size_t)1, std::min({(size_t)2048 / rows, cdiv(places, 1024), (size_t)SCORE_MAX_PARTS}));
  L.wide = places / parts > 4096;
  const size_t step = L.wide ? 4096 : 1024;
  L.part_len = (int64_t)(cdiv(places, parts * step) * step);
  L.parts = (int)cdiv(places, (size_t)L.part_len);
  if (L.parts > 1) {
    const size_t n = rows * L.parts;
    L.off_v = n * sizeof(ScorePart);
    L.off_i = L.off_v + cdiv(n * k * 4, 16) * 16;
    L.bytes = L.off_i + cdiv(n * k * 4, 16) * 16;
  }
  return L;
}

struct ScoreCall {
  const void *logits;
  int64_t ld;
  int n;
  size_t rows;
  ScoreOut o;
  char *ws;
};

template <class E>
static int launch_score(const ScoreCall &c, const ScorePlan &L, hipStream_t s) {
  const auto *x = (const typename E::T *)c.logits;
  ScorePart *ps = (ScorePart *)c.ws;
  float *pv = (float *)(c.ws + L.off_v);
  int *pi = (int *)(c.ws + L.off_i);
  constexpr int V = 16 / sizeof(typename E::T);
  const dim3 grid((unsigned)(c.rows * L.parts));
  if (L.wide)
    hipLaunchKernelGGL((k_score<E, 4, 2>), grid, dim3(128), 0, s, x, c.ld, c.n, L.parts, L.part_len, c.o, ps, pv, pi);
  else
    hipLaunchKernelGGL((k_score<E, 16 / V, 1>), grid, dim3(64), 0, s, x, c.ld, c.n, L.parts, L.part_len, c.o, ps, pv, pi);
  SERVE_TRY(launched("k_score"));
  if (L.parts == 1) return RW_OK;
#define RW_JOIN(K)                                                                                                   \
  hipLaunchKernelGGL((k_score_join<E, K>), dim3((unsigned)c.rows), dim3(256), 0, s, x, c.ld, c.n, L.parts, c.o, ps, pv, pi)
  if (c.o.k <= SCORE_HEADS) RW_JOIN(1);
  else if (c.o.k <= 16) RW_JOIN(16);
  else RW_JOIN(32);
#undef RW_JOIN
  return launched("k_score_join");
}

// --------------------------------------------------------- 8-bit writes

template <class E>
static int launch_write8_of(const PagedView &w, const float *k, size_t ldk, const float *v, size_t ldv, size_t rows,
                            const int32_t *pos, hipStream_t s) {
  const size_t most = MOST_ROWS / w.heads * K8_ROWS;  // rows of one launch
  for (size_t row0 = 0; row0 < rows; row0 += most) {
    const size_t tiles = cdiv(std::min(most, rows - row0), K8_ROWS) * w.heads;
    const dim3 grid((unsigned)cdiv(tiles, 8) * 8);
#define RW_WRITE8(DH)                                                                                              \
  hipLaunchKernelGGL((k_kv_write8<E, DH>), grid, dim3(256), 0, s, w, k, (int64_t)ldk, v, (int64_t)ldv, (int)rows, pos, \
                     (int)tiles, (int)row0)
    switch (w.dim) {
      case 32: RW_WRITE8(32); break;
      case 64: RW_WRITE8(64); break;
      case 96: RW_WRITE8(96); break;
      default: RW_WRITE8(128); break;
    }
#undef RW_WRITE8
    SERVE_TRY(launched("k_kv_write8"));
  }
  return RW_OK;
}

static int launch_write8(int dtype, const PagedView &w, const float *k, size_t ldk, const float *v, size_t ldv, size_t rows,
                         const int32_t *pos, hipStream_t s) {
  return dtype == RW_I8 ? launch_write8_of<I8>(w, k, ldk, v, ldv, rows, pos, s)
                        : launch_write8_of<E4M3>(w, k, ldk, v, ldv, rows, pos, s);
}

template <class E, int ROWS>
static int launch_read_of(const PagedView &w, float *k, size_t ldk, float *v, size_t ldv, size_t rows, const int32_t *pos, hipStream_t s) {
  const size_t most = MOST_ROWS / w.heads * ROWS;  // rows of one launch
  for (size_t row0 = 0; row0 < rows; row0 += most) {
    const size_t tiles = cdiv(std::min(most, rows - row0), ROWS) * w.heads;
    const dim3 grid((unsigned)cdiv(tiles, 8) * 8);
#define RW_READ(DH)                                                                                                    \
  hipLaunchKernelGGL((k_kv_read<E, DH, ROWS>), grid, dim3(256), 0, s, w, k, (int64_t)ldk, v, (int64_t)ldv, (int)rows, pos, \
                     (int)tiles, (int)row0)
    switch (w.dim) {
      case 32: RW_READ(32); break;
      case 64: RW_READ(64); break;
      case 96: RW_READ(96); break;
      default: RW_READ(128); break;
    }
#undef RW_READ
    SERVE_TRY(launched("k_kv_read"));
  }
  return RW_OK;
}

// (ROWS = 64 where that still fills the device: see k_kv_read)
template <class E>
static int launch_read(const PagedView &w, float *k, size_t ldk, float *v, size_t ldv, size_t rows, const int32_t *pos, hipStream_t s) {
  return rows * w.heads >= ((size_t)1 << 17) ? launch_read_of<E, 64>(w, k, ldk, v, ldv, rows, pos, s)
                                             : launch_read_of<E, 32>(w, k, ldk, v, ldv, rows, pos, s);
}

// ----------------------------------------------------------------- book

struct rw_kv_book {
  KvBook b;
};

static int book_fail(BookError e, const char *what) {
  switch (e) {
    case BookError::none: return RW_OK;
    case BookError::seq: return fail(RW_EINVAL, "%s: no such sequence", what);
    case BookError::twice: return fail(RW_EINVAL, "%s: a sequence is listed twice", what);
    case BookError::length: return fail(RW_EINVAL, "%s: length out of range", what);
    case BookError::pages: return fail(RW_ENOMEM, "%s: not enough free pages", what);
    case BookError::seqs: return fail(RW_ENOMEM, "%s: all sequences are in use", what);
    case BookError::room: return fail(RW_EINVAL, "%s: the arrays are too short", what);
  }
  return RW_EINVAL;
}

// a book call that allocates host memory
template <class F>
static int book_call(const char *what, F f) {
  try {
    return book_fail(f(), what);
  } catch (const std::bad_alloc &) {
  } catch (const std::length_error &) {
  }
  return fail(RW_ENOMEM, "%s: host memory exhausted", what);
}

// -------------------------------------------------------------- entries

extern "C" {

int rw_rocm_kv_write_dev(const rw_kv_pages *pages, size_t layer, const float *k, size_t ldk, const float *v, size_t ldv,
                         size_t rows, const int32_t *table, size_t ld_table, size_t n_seqs, const int32_t *seq,
                         const int32_t *pos, void *stream) {
  SERVE_TRY(check_pages(pages));
  if (layer >= pages->n_layer) return fail(RW_EINVAL, "layer %zu of %zu", layer, pages->n_layer);
  if (rows == 0) return RW_OK;
  if (rows > MOST_ROWS) return fail(RW_EINVAL, "rows = %zu: at most %zu", rows, MOST_ROWS);
  const size_t n = (size_t)pages->n_head * pages->head_size;
  SERVE_TRY(check_rows(k, ldk, n, "k"));
  SERVE_TRY(check_rows(v, ldv, n, "v"));
  SERVE_TRY(check_table(table, ld_table, n_seqs, rows, seq, pos, "pos"));
  int dev;
  SERVE_TRY(call_device(pages->k, "the pages' k", &dev));
  const PagedView w = paged_view(pages, layer, table, ld_table, n_seqs, seq);
  if (scaled(pages->dtype)) return launch_write8(pages->dtype, w, k, ldk, v, ldv, rows, pos, (hipStream_t)stream);
  const size_t cols = cdiv(n, KV_COLS), most = MOST_ROWS / cols * KV_ROWS;  // rows of one launch
  for (size_t row0 = 0; row0 < rows; row0 += most) {
    const size_t tiles = cdiv(std::min(most, rows - row0), KV_ROWS) * cols;
    const dim3 grid((unsigned)cdiv(tiles, 8) * 8);
#define RW_WRITE(E)                                                                                                \
  hipLaunchKernelGGL((k_kv_write<E>), grid, dim3(256), 0, (hipStream_t)stream, w, k, (int64_t)ldk, v, (int64_t)ldv, \
                     (int)rows, pos, (int)cols, (int)tiles, (int)row0)
    BY_TYPE(pages->dtype, RW_WRITE);
#undef RW_WRITE
    SERVE_TRY(launched("k_kv_write"));
  }
  return RW_OK;
}

int rw_rocm_kv_read_dev(const rw_kv_pages *pages, size_t layer, float *k, size_t ldk, float *v, size_t ldv, size_t rows,
                        const int32_t *table, size_t ld_table, size_t n_seqs, const int32_t *seq, const int32_t *pos,
                        void *stream) {
  SERVE_TRY(check_pages(pages));
  if (layer >= pages->n_layer) return fail(RW_EINVAL, "layer %zu of %zu", layer, pages->n_layer);
  if (rows == 0) return RW_OK;
  if (rows > MOST_ROWS) return fail(RW_EINVAL, "rows = %zu: at most %zu", rows, MOST_ROWS);
  const size_t n = (size_t)pages->n_head * pages->head_size;
  SERVE_TRY(check_rows(k, ldk, n, "k"));
  SERVE_TRY(check_rows(v, ldv, n, "v"));
  SERVE_TRY(check_table(table, ld_table, n_seqs, rows, seq, pos, "pos"));
  int dev;
  SERVE_TRY(call_device(pages->k, "the pages' k", &dev));
  const PagedView w = paged_view(pages, layer, table, ld_table, n_seqs, seq);
#define RW_READ(E) SERVE_TRY(launch_read<E>(w, k, ldk, v, ldv, rows, pos, (hipStream_t)stream))
  if (pages->dtype == RW_I8) RW_READ(I8);
  else if (pages->dtype == RW_E4M3) RW_READ(E4M3);
  else BY_TYPE(pages->dtype, RW_READ);
#undef RW_READ
  return RW_OK;
}

// every id in the pool, no dst twice, no dst a src
static int check_copies(const rw_kv_pages *p, const int32_t *src, const int32_t *dst, size_t n) {
  for (size_t i = 0; i < n; ++i)
    if (src[i] < 0 || (size_t)src[i] >= p->n_pages || dst[i] < 0 || (size_t)dst[i] >= p->n_pages)
      return fail(RW_EINVAL, "copy %zu: page %d -> %d of %zu", i, src[i], dst[i], p->n_pages);
  std::vector<int32_t> d(dst, dst + n);
  std::sort(d.begin(), d.end());
  for (size_t i = 1; i < n; ++i)
    if (d[i] == d[i - 1]) return fail(RW_EINVAL, "page %d is written twice", d[i]);
  for (size_t i = 0; i < n; ++i)
    if (std::binary_search(d.begin(), d.end(), src[i])) return fail(RW_EINVAL, "page %d is read and written", src[i]);
  return RW_OK;
}

int rw_rocm_kv_copy_pages_dev(const rw_kv_pages *pages, const int32_t *src, const int32_t *dst, size_t n, void *stream) {
  SERVE_TRY(check_pages(pages));
  if (n == 0) return RW_OK;
  if (!src || !dst) return fail(RW_EINVAL, "src or dst is NULL");
  if (n > pages->n_pages) return fail(RW_EINVAL, "%zu copies in a pool of %zu pages", n, pages->n_pages);
  try {
    SERVE_TRY(check_copies(pages, src, dst, n));
  } catch (const std::bad_alloc &) {
    return fail(RW_ENOMEM, "host memory exhausted");
  }
  int dev;
  SERVE_TRY(call_device(pages->k, "the pages' k", &dev));
  const size_t page_rows = (size_t)pages->n_head * pages->page_rows;  // of one head
  const size_t piece = page_rows * pages->head_size * pool_size(pages->dtype) / 16;
  for (size_t i0 = 0; i0 < n; i0 += KV_PAIRS) {
    const size_t m = std::min((size_t)KV_PAIRS, n - i0);
    KvPairs pairs{};
    for (size_t i = 0; i < m; ++i) pairs.id[i] = make_int2(src[i0 + i], dst[i0 + i]);
    hipLaunchKernelGGL(k_kv_copy, dim3((unsigned)cdiv(piece, 256), (unsigned)m, (unsigned)(2 * pages->n_layer)),
                       dim3(256), 0, (hipStream_t)stream, (uint4 *)pages->k, (uint4 *)pages->v, (int64_t)piece,
                       (int64_t)pages->n_pages, pairs);
    SERVE_TRY(launched("k_kv_copy"));
    if (!scaled(pages->dtype)) continue;
    hipLaunchKernelGGL(k_kv_copy, dim3((unsigned)cdiv(page_rows / 4, 256), (unsigned)m, (unsigned)(2 * pages->n_layer)),
                       dim3(256), 0, (hipStream_t)stream, (uint4 *)pages->k_scale, (uint4 *)pages->v_scale,
                       (int64_t)(page_rows / 4), (int64_t)pages->n_pages, pairs);
    SERVE_TRY(launched("k_kv_copy"));
  }
  return RW_OK;
}

size_t rw_rocm_paged_attention_workspace_size(const rw_kv_pages *pages, size_t rows, int n_head, size_t max_len) {
  if (check_pages(pages) || check_paged_heads(pages, rows, n_head, max_len) || rows == 0) return 0;
  if (scaled(pages->dtype)) return tree_workspace(pages, n_head, rows, rows, 1, max_len);
  return paged_bytes(paged_plan(pages, rows, n_head, max_len), rows, n_head, pages->head_size);
}

int rw_rocm_paged_attention_dev(const rw_kv_pages *pages, size_t layer, const float *q, size_t ldq, size_t rows,
                                int n_head, const int32_t *table, size_t ld_table, size_t n_seqs, const int32_t *seq,
                                const int32_t *len, size_t max_len, float *out, size_t ldo, void *workspace,
                                size_t workspace_len, void *stream) {
  SERVE_TRY(check_pages(pages));
  if (layer >= pages->n_layer) return fail(RW_EINVAL, "layer %zu of %zu", layer, pages->n_layer);
  SERVE_TRY(check_paged_heads(pages, rows, n_head, max_len));
  if (rows == 0) return RW_OK;
  const size_t n = (size_t)n_head * pages->head_size;
  SERVE_TRY(check_rows(q, ldq, n, "q"));
  SERVE_TRY(check_rows(out, ldo, n, "out"));
  SERVE_TRY(check_table(table, ld_table, n_seqs, rows, seq, len, "len"));
  int dev;
  SERVE_TRY(call_device(pages->k, "the pages' k", &dev));
  if (scaled(pages->dtype)) {
    CallWorkspace hold;
    void *ws = nullptr;
    SERVE_TRY(hold.take(dev, workspace, workspace_len, tree_workspace(pages, n_head, rows, rows, 1, max_len), stream, &ws));
    return tree_launch(TreeCall{paged_view(pages, layer, table, ld_table, n_seqs, seq), pages->dtype, q, (int64_t)ldq, rows,
                                n_head, rows, nullptr, len, 1, nullptr, 0, max_len, out, (int64_t)ldo},
                       pages, ws, (hipStream_t)stream);
  }
  PagedCall c{paged_view(pages, layer, table, ld_table, n_seqs, seq), q, (int64_t)ldq, (int)rows, n_head, 0, len, out,
              (int64_t)ldo, nullptr};
  c.max_len = (int)std::min(max_len, std::min((size_t)1 << 30, ld_table * pages->page_rows));
  const PagedPlan L = paged_plan(pages, rows, n_head, (size_t)c.max_len);
  // told by max_len alone, so that the size does not depend on the table's width
  const size_t need = workspace ? rw_rocm_paged_attention_workspace_size(pages, rows, n_head, max_len)
                                : paged_bytes(L, rows, n_head, pages->head_size);
  CallWorkspace hold;
  void *ws = nullptr;
  SERVE_TRY(hold.take(dev, workspace, workspace_len, need, stream, &ws));
  c.part = (float *)ws;
  hipStream_t s = (hipStream_t)stream;
  switch (pages->dtype) {
    case RW_F32: return launch_paged_dim<F32>(c, L, s);
    case RW_F16: return launch_paged_dim<F16>(c, L, s);
    default: return launch_paged_dim<BF16>(c, L, s);
  }
}

int rw_rocm_kv_book_create(size_t n_pages, size_t page_rows, size_t max_seqs, rw_kv_book **out) {
  if (!out) return fail(RW_EINVAL, "out is NULL");
  *out = nullptr;
  if (n_pages < 1 || n_pages > (size_t)INT32_MAX) return fail(RW_EINVAL, "n_pages %zu: between 1 and 2^31 - 1", n_pages);
  if (page_rows < 16 || page_rows > 256 || (page_rows & (page_rows - 1)))
    return fail(RW_EINVAL, "page_rows %zu: 16, 32, 64, 128 or 256", page_rows);
  if (max_seqs < 1 || max_seqs > (size_t)INT32_MAX) return fail(RW_EINVAL, "max_seqs %zu: between 1 and 2^31 - 1", max_seqs);
  return book_call("kv_book_create", [&] {
    *out = new rw_kv_book{KvBook(n_pages, page_rows, max_seqs)};
    return BookError::none;
  });
}

void rw_rocm_kv_book_free(rw_kv_book *b) { delete b; }

int rw_rocm_kv_book_add(rw_kv_book *b, size_t n, int32_t *seqs) {
  if (!b || (n && !seqs)) return fail(RW_EINVAL, "book or seqs is NULL");
  return book_call("kv_book_add", [&] { return b->b.add(n, seqs); });
}

int rw_rocm_kv_book_fork(rw_kv_book *b, const int32_t *from, size_t n, int32_t *seqs) {
  if (!b || (n && (!from || !seqs))) return fail(RW_EINVAL, "book, from or seqs is NULL");
  return book_call("kv_book_fork", [&] { return b->b.fork(from, n, seqs); });
}

int rw_rocm_kv_book_extend(rw_kv_book *b, const int32_t *seqs, size_t n, const size_t *more, int32_t *src, int32_t *dst,
                           size_t *n_copies) {
  if (!b || !n_copies || (n && (!seqs || !more || !src || !dst)))
    return fail(RW_EINVAL, "book, seqs, more, src, dst or n_copies is NULL");
  return book_call("kv_book_extend", [&] { return b->b.extend(seqs, n, more, src, dst, n_copies); });
}

int rw_rocm_kv_book_truncate(rw_kv_book *b, int32_t seq, size_t len) {
  if (!b) return fail(RW_EINVAL, "book is NULL");
  return book_fail(b->b.truncate(seq, len), "kv_book_truncate");
}

int rw_rocm_kv_book_release(rw_kv_book *b, const int32_t *seqs, size_t n) {
  if (!b || (n && !seqs)) return fail(RW_EINVAL, "book or seqs is NULL");
  return book_fail(b->b.release(seqs, n), "kv_book_release");
}

int rw_rocm_kv_book_compact(rw_kv_book *b, int32_t *src, int32_t *dst, size_t cap, size_t *n) {
  if (!b || !n || (cap && (!src || !dst))) return fail(RW_EINVAL, "book, src, dst or n is NULL");
  return book_call("kv_book_compact", [&] { return b->b.compact(src, dst, cap, n); });
}

int rw_rocm_kv_book_table(const rw_kv_book *b, const int32_t *seqs, size_t n, int32_t *table, size_t ld) {
  if (!b || (n && (!seqs || !table))) return fail(RW_EINVAL, "book, seqs or table is NULL");
  for (size_t i = 0; i < n; ++i) {
    if (!b->b.live(seqs[i])) return book_fail(BookError::seq, "kv_book_table");
    if (b->b.pages(seqs[i]).size() > ld)
      return fail(RW_EINVAL, "sequence %d has %zu pages, a table row %zu", seqs[i], b->b.pages(seqs[i]).size(), ld);
  }
  for (size_t i = 0; i < n; ++i) {
    const std::vector<int32_t> &p = b->b.pages(seqs[i]);
    std::copy(p.begin(), p.end(), table + i * ld);
    std::fill(table + i * ld + p.size(), table + (i + 1) * ld, 0);
  }
  return RW_OK;
}

int rw_rocm_kv_book_len(const rw_kv_book *b, int32_t seq, size_t *len) {
  if (!b || !len) return fail(RW_EINVAL, "book or len is NULL");
  if (!b->b.live(seq)) return book_fail(BookError::seq, "kv_book_len");
  *len = b->b.len(seq);
  return RW_OK;
}

int rw_rocm_kv_book_info(const rw_kv_book *b, size_t *free_pages, size_t *used_pages, size_t *n_seqs) {
  if (!b) return fail(RW_EINVAL, "book is NULL");
  if (free_pages) *free_pages = b->b.free_pages();
  if (used_pages) *used_pages = b->b.n_pages() - b->b.free_pages();
  if (n_seqs) *n_seqs = b->b.n_seqs();
  return RW_OK;
}

size_t rw_rocm_token_logprobs_workspace_size(size_t rows, size_t n_vocab, size_t k) {
  if (rows == 0 || rows > MOST_ROWS || n_vocab == 0 || n_vocab > (size_t)INT32_MAX || k > (size_t)SCORE_TOP) return 0;
  return score_plan(rows, n_vocab, k).bytes;
}

int rw_rocm_token_logprobs_dev(int dtype, const void *logits, size_t ld, size_t rows, size_t n_vocab,
                               const uint32_t *tokens, size_t n_tok, float *logprobs, float *entropy, size_t k,
                               uint32_t *top_ids, float *top_logprobs, void *workspace, size_t workspace_len,
                               void *stream) {
  if (!elem_size(dtype)) return fail(RW_EINVAL, "unsupported dtype %d (RW_F32, RW_F16 or RW_BF16)", dtype);
  if (k > (size_t)SCORE_TOP) return fail(RW_EINVAL, "k = %zu: at most %d", k, SCORE_TOP);
  if (n_vocab < 1 || n_vocab > (size_t)INT32_MAX) return fail(RW_EINVAL, "n_vocab = %zu: between 1 and 2^31 - 1", n_vocab);
  if (rows > MOST_ROWS || n_tok > (size_t)INT32_MAX) return fail(RW_EINVAL, "rows = %zu, n_tok = %zu", rows, n_tok);
  if (rows == 0) return RW_OK;
  if (!logits || !aligned(logits, elem_size(dtype))) return fail(RW_EINVAL, "logits is NULL or not aligned");
  if (ld < n_vocab || ld > ((size_t)1 << 40)) return fail(RW_EINVAL, "logits: row stride %zu for rows of %zu", ld, n_vocab);
  if (n_tok && (!tokens || !logprobs)) return fail(RW_EINVAL, "tokens or logprobs is NULL");
  if (k && (!top_ids || !top_logprobs)) return fail(RW_EINVAL, "top_ids or top_logprobs is NULL");
  if (!aligned(tokens, 4) || !aligned(logprobs, 4) || !aligned(entropy, 4) || !aligned(top_ids, 4) || !aligned(top_logprobs, 4))
    return fail(RW_EINVAL, "tokens and results must be 4-byte aligned");
  int dev;
  SERVE_TRY(call_device(logits, "logits", &dev));
  const ScorePlan L = score_plan(rows, n_vocab, k);
  CallWorkspace hold;
  void *ws = nullptr;
  SERVE_TRY(hold.take(dev, workspace, workspace_len, L.bytes, stream, &ws));
  const ScoreCall c{logits, (int64_t)ld, (int)n_vocab, rows,
                    ScoreOut{tokens, logprobs, entropy, top_ids, top_logprobs, (int64_t)n_tok, (int)k}, (char *)ws};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case RW_F32: return launch_score<F32>(c, L, s);
    case RW_F16: return launch_score<F16>(c, L, s);
    default: return launch_score<BF16>(c, L, s);
  }
}

}  // extern "C"
