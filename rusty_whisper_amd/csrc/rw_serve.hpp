// rw_serve.hpp -- what the serving entries' translation units share: the checks
// of their arguments and the workspace of a call (host code).
#pragma once
#include <hip/hip_runtime.h>

#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

#include "rw_internal.hpp"
#include "rw_kv.hpp"
#include "rw_rocm.h"

namespace rw {

inline int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return rw_internal_fail(code, buf);
}

#define SERVE_TRY(expr)  \
  do {                   \
    int rc_ = (expr);    \
    if (rc_) return rc_; \
  } while (0)

inline int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RW_OK : fail(RW_EHIP, "launch of %s: %s", what, hipGetErrorString(e));
}

inline size_t cdiv(size_t a, size_t b) { return (a + b - 1) / b; }
inline bool aligned(const void *p, size_t a) { return (uintptr_t)p % a == 0; }

// rows (times heads) of one call: a workgroup of 256 threads each stays below
// the 2^32 threads a launch may have
constexpr size_t MOST_ROWS = (size_t)1 << 23;

// bytes of a logit, 0: not a type of logits
inline int elem_size(int dtype) { return dtype == RW_F32 ? 4 : dtype == RW_F16 || dtype == RW_BF16 ? 2 : 0; }
// bytes of a pool's value, 0: not a type of pools
inline bool scaled(int dtype) { return dtype == RW_I8 || dtype == RW_E4M3; }
inline int pool_size(int dtype) { return scaled(dtype) ? 1 : elem_size(dtype); }

// The current device, which has to hold `p` (an array of the call; `what`
// names it): kernels that ran elsewhere would fault on it.
inline int call_device(const void *p, const char *what, int *dev) {
  SERVE_TRY(rw_internal_current_device(dev));
  hipPointerAttribute_t at{};
  if (hipPointerGetAttributes(&at, p) != hipSuccess) {
    (void)hipGetLastError();
    return fail(RW_EINVAL, "%s is not device memory", what);
  }
  if (at.type == hipMemoryTypeUnregistered || at.type == hipMemoryTypeHost)
    return fail(RW_EINVAL, "%s is not device memory", what);
  if (at.type == hipMemoryTypeDevice && at.device != *dev)
    return fail(RW_EINVAL, "%s is on device %d, the current device is %d", what, at.device, *dev);
  return RW_OK;
}

inline int check_pages(const rw_kv_pages *p) {
  if (!p) return fail(RW_EINVAL, "pages is NULL");
  if (!pool_size(p->dtype))
    return fail(RW_EINVAL, "unsupported dtype %d (RW_F32, RW_F16, RW_BF16, RW_I8 or RW_E4M3)", p->dtype);
  if (p->head_size != 32 && p->head_size != 64 && p->head_size != 96 && p->head_size != 128)
    return fail(RW_EINVAL, "head_size %d: 32, 64, 96 or 128", p->head_size);
  if (p->page_rows < 16 || p->page_rows > 256 || (p->page_rows & (p->page_rows - 1)))
    return fail(RW_EINVAL, "page_rows %d: 16, 32, 64, 128 or 256", p->page_rows);
  if (p->n_head < 1 || p->n_head > 65535) return fail(RW_EINVAL, "n_head %d: between 1 and 65535", p->n_head);
  if (p->n_layer < 1 || p->n_layer > 32767) return fail(RW_EINVAL, "n_layer %zu: between 1 and 32767", p->n_layer);
  if (p->n_pages < 1 || p->n_pages > (size_t)INT32_MAX) return fail(RW_EINVAL, "n_pages %zu: between 1 and 2^31 - 1", p->n_pages);
  if (!p->k || !p->v || !aligned(p->k, 16) || !aligned(p->v, 16))
    return fail(RW_EINVAL, "the pages' k and v must be 16-byte aligned device memory");
  if (scaled(p->dtype) && (!p->k_scale || !p->v_scale || !aligned(p->k_scale, 16) || !aligned(p->v_scale, 16)))
    return fail(RW_EINVAL, "the pages' k_scale and v_scale must be 16-byte aligned device memory");
  return RW_OK;
}

inline int check_rows(const float *a, size_t ld, size_t n, const char *what) {
  if (!a) return fail(RW_EINVAL, "%s is NULL", what);
  if (ld < n || ld > ((size_t)1 << 40)) return fail(RW_EINVAL, "%s: row stride %zu for rows of %zu", what, ld, n);
  if (ld % 4 || !aligned(a, 16)) return fail(RW_EINVAL, "%s rows must be 16-byte aligned", what);
  return RW_OK;
}

inline int check_table(const int32_t *table, size_t ld, size_t n_seqs, size_t rows, const int32_t *seq, const int32_t *at,
                       const char *what) {
  if (!table || !at) return fail(RW_EINVAL, "%s is NULL", table ? what : "table");
  if (!aligned(table, 4) || !aligned(seq, 4) || !aligned(at, 4)) return fail(RW_EINVAL, "index arrays must be 4-byte aligned");
  if (ld < 1 || n_seqs < 1 || ld > (size_t)INT32_MAX || n_seqs > (size_t)INT32_MAX)
    return fail(RW_EINVAL, "a table of %zu sequences and %zu pages each", n_seqs, ld);
  if (!seq && rows > n_seqs) return fail(RW_EINVAL, "%zu rows for a table of %zu sequences, and no seq", rows, n_seqs);
  return RW_OK;
}

inline int check_paged_heads(const rw_kv_pages *p, size_t rows, int n_head, size_t max_len) {
  if (n_head < 1 || n_head % p->n_head)
    return fail(RW_EINVAL, "n_head %d is not a positive multiple of the pages' %d", n_head, p->n_head);
  if (rows > MOST_ROWS / n_head) return fail(RW_EINVAL, "%zu rows of %d heads", rows, n_head);
  if (max_len > (size_t)INT32_MAX) return fail(RW_EINVAL, "max_len %zu", max_len);
  return RW_OK;
}

inline PagedView paged_view(const rw_kv_pages *p, size_t layer, const int32_t *table, size_t ld, size_t n_seqs,
                            const int32_t *seq) {
  const size_t rows = layer * p->n_pages * p->n_head * p->page_rows, off = rows * p->head_size * pool_size(p->dtype);
  const bool s = scaled(p->dtype);
  return PagedView{(const char *)p->k + off, (const char *)p->v + off, p->n_head, p->head_size,
                   __builtin_ctz((unsigned)p->page_rows), (int)p->n_pages, table, (int)n_seqs, (int64_t)ld, seq,
                   s ? p->k_scale + rows : nullptr, s ? p->v_scale + rows : nullptr};
}

// calls CALL(E) for the element type of `dtype`
#define BY_TYPE(dtype, CALL)               \
  do {                                     \
    if ((dtype) == RW_F32) CALL(F32);      \
    else if ((dtype) == RW_F16) CALL(F16); \
    else CALL(BF16);                       \
  } while (0)

// The workspace of a call: the caller's, or this stream's.  A stream that is
// being captured has to bring one: the library's may be replaced by a later
// call while the graph still uses it.
struct CallWorkspace {
  void *slot = nullptr;
  CallWorkspace() = default;
  CallWorkspace(const CallWorkspace &) = delete;
  CallWorkspace &operator=(const CallWorkspace &) = delete;
  ~CallWorkspace() {
    if (slot) rw_internal_workspace_release(slot);
  }
  int take(int dev, void *given, size_t len, size_t need, void *stream, void **out) {
    *out = given;
    if (need == 0) return RW_OK;
    if (given) {
      if (len < need) return fail(RW_EINVAL, "workspace of %zu bytes < %zu needed", len, need);
      if (!aligned(given, 16)) return fail(RW_EINVAL, "the workspace must be 16-byte aligned");
      return RW_OK;
    }
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    const hipError_t e = hipStreamIsCapturing((hipStream_t)stream, &st);
    if (e != hipSuccess) return fail(RW_EHIP, "hipStreamIsCapturing: %s", hipGetErrorString(e));
    if (st != hipStreamCaptureStatusNone) return fail(RW_EINVAL, "a captured call needs a workspace of %zu bytes", need);
    return rw_internal_workspace(dev, stream, need, &slot, out);
  }
};

// ------------------------------------------- attention of several new rows

// One call of the attention that rw_tree.hpp has kernels for (rw_draft.hip).
// starts null: tree i is row i alone and sees the first past[i] rows.
struct TreeCall {
  PagedView w;
  int dtype;
  const float *q;
  int64_t ldq;
  size_t rows;
  int n_head;
  size_t n_trees;
  const int32_t *starts, *past;
  size_t max_rows;
  const uint32_t *mask;
  int n_words;
  size_t max_len;
  float *out;
  int64_t ldo;
};
// Bytes of its workspace; never falls with max_len.
size_t tree_workspace(const rw_kv_pages *pages, int n_head, size_t rows, size_t n_trees, size_t max_rows, size_t max_len);
int tree_launch(const TreeCall &c, const rw_kv_pages *pages, void *ws, hipStream_t s);

}  // namespace rw
