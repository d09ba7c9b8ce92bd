// mi_paged.hpp -- device view of a paged K/V cache and of the sequences of one call, shared by
// the append (mi_rope.hip) and the attention (mi_paged.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mi_host.hpp"

namespace mig {

struct PagedView {
  const int32_t* q_start;  // null: one new token for each sequence
  const int32_t* kv_len;
  const int32_t* pages;
  int64_t pages_ld;
  int64_t page_stride, head_stride, slot_stride;  // elements
  int n_seqs, total_q, max_pages, num_pages, page_shift;
};

// Rows [q0, q0 + n) of sequence s among the call's rows, cut to them whatever q_start holds.
__device__ __forceinline__ void seq_rows(const PagedView& v, int s, int& q0, int& n) {
  if (!v.q_start) {
    q0 = s;
    n = 1;
    return;
  }
  const int a = min(max(v.q_start[s], 0), v.total_q), b = min(max(v.q_start[s + 1], 0), v.total_q);
  q0 = a;
  n = max(b - a, 0);
}

// The page of position pos of sequence s, -1 if there is none.
__device__ __forceinline__ int page_of(const PagedView& v, int s, int64_t pos) {
  const int64_t i = pos >> v.page_shift;
  if (pos < 0 || i >= v.max_pages) return -1;
  const int page = v.pages[(int64_t)s * v.pages_ld + i];
  return (uint32_t)page < (uint32_t)v.num_pages ? page : -1;
}

// First k in [0, n) at which below(k) is false, n if there is none; below must be true up to there
// and false from there on.  The whole wave searches with one k per lane, 64-fold a step; whatever
// below answers, it ends with a value in [0, n].
template <class F>
__device__ __forceinline__ int wave_first_false(int n, F below) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int step = (hi - lo + 63) >> 6;
    const int64_t k = lo + (int64_t)lane * step;
    const bool b = k < hi && below((int)k);
    const int c = __popcll(__ballot(b));
    if (c == 0) break;
    const int64_t end = lo + (int64_t)c * step;
    lo += (c - 1) * step + 1;
    hi = end < hi ? (int)end : hi;
  }
  return lo;
}

// Checks cache and seqs of an entry point; MI_OK or an error with its text.
inline int check_paged(const mi_paged_cache* c, const mi_paged_seqs* s) {
  if (!c || !s) return host_fail(MI_ERR_NULL, "cache or seqs is NULL");
  if (s->n_seqs < 0 || s->total_q < 0 || s->max_pages < 0 || c->num_pages < 0 || c->n_kv < 0 || c->head_dim < 0)
    return host_fail(MI_ERR_SHAPE, "negative size");
  if (s->n_seqs > INT32_MAX || s->total_q > INT32_MAX || s->max_pages > INT32_MAX || c->num_pages > INT32_MAX ||
      c->n_kv > INT32_MAX)
    return host_fail(MI_ERR_SHAPE, "size exceeds 2^31-1");
  if (c->page_size < 1 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)))
    return host_fail(MI_ERR_SHAPE, "page_size=%lld is not a power of two up to 2^20", (long long)c->page_size);
  if (!s->q_start && s->total_q != s->n_seqs)
    return host_fail(MI_ERR_SHAPE, "total_q=%lld for %lld sequences without q_start", (long long)s->total_q,
                     (long long)s->n_seqs);
  if (s->max_pages * c->page_size > INT32_MAX - 4096)
    return host_fail(MI_ERR_SHAPE, "max_pages * page_size = %lld exceeds 2^31 - 4096",
                     (long long)(s->max_pages * c->page_size));
  if (s->pages_ld < s->max_pages)
    return host_fail(MI_ERR_LD, "pages_ld=%lld < max_pages=%lld", (long long)s->pages_ld, (long long)s->max_pages);
  if (s->n_seqs == 0 || s->total_q == 0) return MI_OK;
  if (!s->kv_len || (s->max_pages > 0 && !s->pages)) return host_fail(MI_ERR_NULL, "kv_len or pages is NULL");
  if (((uintptr_t)s->q_start | (uintptr_t)s->kv_len | (uintptr_t)s->pages) & 3)
    return host_fail(MI_ERR_UNSUPPORTED, "q_start, kv_len and pages must be aligned to their element size");
  if (c->num_pages > 0 && (!c->k || !c->v)) return host_fail(MI_ERR_NULL, "cache k or v is NULL");
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15)
    return host_fail(MI_ERR_UNSUPPORTED, "cache k and v must be 16-byte aligned");
  if (c->head_dim < 8 || c->head_dim % 8)
    return host_fail(MI_ERR_UNSUPPORTED, "head_dim %lld: a multiple of 8 is needed", (long long)c->head_dim);
  if ((c->page_stride | c->head_stride | c->slot_stride) % 8)
    return host_fail(MI_ERR_UNSUPPORTED, "cache strides must be multiples of 8 elements");
  if ((c->page_size > 1 && c->slot_stride < c->head_dim) || (c->n_kv > 1 && c->head_stride < c->head_dim) ||
      (c->num_pages > 1 && c->page_stride < c->head_dim))
    return host_fail(MI_ERR_LD, "a cache stride is shorter than a row of %lld", (long long)c->head_dim);
  return MI_OK;
}

inline PagedView paged_view(const mi_paged_cache* c, const mi_paged_seqs* s) {
  PagedView v;
  v.q_start = s->q_start;
  v.kv_len = s->kv_len;
  v.pages = s->pages;
  v.pages_ld = s->pages_ld;
  v.page_stride = c->page_stride;
  v.head_stride = c->head_stride;
  v.slot_stride = c->slot_stride;
  v.n_seqs = (int)s->n_seqs;
  v.total_q = (int)s->total_q;
  v.max_pages = (int)s->max_pages;
  v.num_pages = (int)c->num_pages;
  v.page_shift = 0;
  while ((int64_t{1} << v.page_shift) < c->page_size) ++v.page_shift;
  return v;
}

}  // namespace mig
