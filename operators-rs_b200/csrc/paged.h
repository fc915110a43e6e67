// paged.h — what the operators of a paged serving batch share: the batch as the kernels see it, its checks, the status words.
#pragma once
#include <atomic>
#include <new>

#include "common.h"
#include "paged_schedule.h"

namespace ops {

// The device arrays of an ops_paged_batch.  Their values are not known on the host: every kernel takes them through the
// functions below, which cut whatever would lead outside the tensors.
struct PagedBatch {
  const uint32_t *table, *start, *len;  // [nseq, width], [nseq + 1], [nseq]
  long long table_ld;                   // elements between the rows of the table
  int nseq, width, nt;
  uint32_t npages, max_seq;             // max_seq: 0xffffffff when unknown
  int page_log2;
  int *status;
};

#ifdef __CUDACC__
// cut to the step's rows; a decreasing or overrunning seq_start is an empty or shorter sequence
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch &b, int i, bool report) {
  const uint32_t nt = (uint32_t)b.nt, raw0 = b.start[i], raw1 = b.start[i + 1], cap = (uint32_t)b.width << b.page_log2;
  const uint32_t raw_len = b.len[i];
  const uint32_t r0 = min(raw0, nt), r1 = max(min(raw1, nt), r0);
  PagedSeq s;
  s.row = (int)r0;
  s.n = (int)(r1 - r0);
  s.len = (int)min(raw_len, cap);
  if (report) {
    if (raw0 > raw1 || raw1 > nt || (uint32_t)s.n > b.max_seq) atomicCAS(b.status, 0, OPS_PAGED_BAD_ROWS);
    if (raw_len > cap) atomicCAS(b.status, 0, OPS_PAGED_BAD_LENGTH);
  }
  return s;
}

// The sequence that owns `row` — the last one that starts at or before it — by one warp, 32 probes a round: a few dependent
// loads instead of log2(nseq).  All lanes get the answer (-1: in front of the first sequence).  Starts that do not ascend give
// some sequence of the batch; the caller checks that the row lies in it.
__device__ __forceinline__ int paged_find(const PagedBatch &b, uint32_t row) {
  const int lane = threadIdx.x & 31;
  int lo = -1, hi = b.nseq;  // start[lo] <= row < start[hi], with start[-1] = -inf, start[nseq] = +inf
  while (hi - lo > 1) {
    const int step = (hi - lo + 32) / 33;
    const int at = lo + (lane + 1) * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && b.start[min(at, b.nseq - 1)] <= row);
    const int k = below == 0xffffffffu ? 32 : __ffs(~below) - 1;  // lanes 0..k-1 without a gap say "at or before"
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}
#endif

// Shapes and types of the batch and the cache; `page_log2` and the merged shape come back when they are static.
struct PagedMeta {
  usz nseq, width, npages, nkvh, page, dh;
  int page_log2;
};

inline int paged_meta(const ops_paged_batch *b, const ops_layout *k, const ops_layout *v, PagedMeta *m) {
  if (b->page_table_layout.ndim != 2) return fail(OPS_RANK_NOT_SUPPORT, "page_table.ndim = %u, 2 expected", b->page_table_layout.ndim);
  if (b->seq_start_layout.ndim != 1) return fail(OPS_RANK_NOT_SUPPORT, "seq_start.ndim = %u, 1 expected", b->seq_start_layout.ndim);
  if (b->kv_len_layout.ndim != 1) return fail(OPS_RANK_NOT_SUPPORT, "kv_len.ndim = %u, 1 expected", b->kv_len_layout.ndim);
  if (k->ndim != 4) return fail(OPS_RANK_NOT_SUPPORT, "k_pages.ndim = %u, 4 expected", k->ndim);
  if (v->ndim != 4) return fail(OPS_RANK_NOT_SUPPORT, "v_pages.ndim = %u, 4 expected", v->ndim);
  const ops_layout *ints[3] = {&b->page_table_layout, &b->seq_start_layout, &b->kv_len_layout};
  static const char *names[3] = {"page_table", "seq_start", "kv_len"};
  for (int i = 0; i < 3; ++i)
    if (ints[i]->dt != OPS_DT_U32 && ints[i]->dt != OPS_DT_I32) return fail(OPS_TYPE_NOT_SUPPORT, "data type of %s is not supported, must be u32 or i32", names[i]);
  usz starts = b->seq_start_layout.shape[0];
  if (!dyn(starts)) {
    if (starts == 0) return fail(OPS_SHAPE_MISMATCH, "seq_start is empty, nseq + 1 entries expected");
    --starts;
  }
  const usz nseqs[3] = {b->page_table_layout.shape[0], b->kv_len_layout.shape[0], starts};
  if (!merge_dims(nseqs, 3, &m->nseq)) return fail(OPS_SHAPE_MISMATCH, "nseq of page_table, kv_len and seq_start (nseq + 1) differ");
  m->width = b->page_table_layout.shape[1];
  const usz np[2] = {k->shape[0], v->shape[0]}, nk[2] = {k->shape[1], v->shape[1]}, pg[2] = {k->shape[2], v->shape[2]}, dh[2] = {k->shape[3], v->shape[3]};
  if (!merge_dims(np, 2, &m->npages)) return fail(OPS_SHAPE_MISMATCH, "npages of k_pages and v_pages differ");
  if (!merge_dims(nk, 2, &m->nkvh)) return fail(OPS_SHAPE_MISMATCH, "nkvh of k_pages and v_pages differ");
  if (!merge_dims(pg, 2, &m->page)) return fail(OPS_SHAPE_MISMATCH, "page size of k_pages and v_pages differ");
  if (!merge_dims(dh, 2, &m->dh)) return fail(OPS_SHAPE_MISMATCH, "dh of k_pages and v_pages differ");
  m->page_log2 = 0;
  if (!dyn(m->page)) {
    if (m->page < 8 || m->page > 65536 || (m->page & (m->page - 1))) return fail(OPS_SHAPE_NOT_SUPPORT, "page size %zu, a power of two from 8 to 65536 expected", m->page);
    while (((usz)1 << m->page_log2) < m->page) ++m->page_log2;
  }
  return OPS_OK;
}

// Everything a launch needs to be static, in range and aligned; fills the device view.
inline int paged_launch_checks(const char *op, const ops_paged_batch *b, const ops_layout *k, const void *k_base, const ops_layout *v, const void *v_base,
                               const PagedMeta &m, usz nt, int *status, PagedBatch *out) {
  if (dyn(m.nseq) || dyn(m.width) || dyn(m.npages) || dyn(m.nkvh) || dyn(m.page) || dyn(m.dh) || dyn(b->page_table_layout.strides[0]) ||
      dyn(b->page_table_layout.strides[1]) || dyn(b->seq_start_layout.strides[0]) || dyn(b->kv_len_layout.strides[0]))
    return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: every shape and stride of the batch and the cache must be static at launch", op);
  if (dyn(b->page_table_layout.shape[0]) || dyn(b->seq_start_layout.shape[0]) || dyn(b->kv_len_layout.shape[0]))
    return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: every shape of the batch must be static at launch", op);
  for (int d = 0; d < 4; ++d)
    if (dyn(k->shape[d]) || dyn(v->shape[d]) || dyn(k->strides[d]) || dyn(v->strides[d])) return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: every shape and stride of the cache must be static at launch", op);
  if ((m.width > 1 && b->page_table_layout.strides[1] != 4) || (m.nseq > 1 && b->page_table_layout.strides[0] % 4) ||
      (m.nseq > 0 && b->seq_start_layout.strides[0] != 4) || (m.nseq > 1 && b->kv_len_layout.strides[0] != 4))
    return fail(OPS_STRIDES_NOT_SUPPORT, "%s: seq_start, kv_len and the rows of page_table must be contiguous", op);
  if (m.nseq > 0x3fffffffu || m.npages > 0x7fffffffu || m.nkvh > 0xffffu || nt > 0x3fffffffu || m.width > 0x3fffffffu ||
      m.width * m.page > 0x3fffffffu)
    return fail(OPS_SHAPE_NOT_SUPPORT, "%s: more than 2^30 rows, sequences or slots of a sequence, or too many pages or heads", op);
  const ops_layout *caches[2] = {k, v};
  const void *bases[2] = {k_base, v_base};
  const usz dims[3] = {m.npages, m.nkvh, m.page};
  for (int i = 0; i < 2; ++i) {
    if (caches[i]->strides[3] != 2) return fail(OPS_STRIDES_NOT_SUPPORT, "%s: last dim of the cache must be contiguous", op);
    for (int d = 0; d < 3; ++d)
      if (dims[d] > 1 && (caches[i]->strides[d] % 16 || caches[i]->strides[d] <= 0 || caches[i]->strides[d] >= ((isz)1 << 36)))
        return fail(OPS_STRIDES_NOT_SUPPORT, "%s: strides of the cache must be multiples of 16 bytes, positive and below 2^36", op);
  }
  if (nt == 0 || m.nseq == 0) return OPS_OK;
  if (!b->seq_start_base || !b->kv_len_base || (m.width && !b->page_table_base))
    return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: null base pointer of the batch at launch", op);
  if (!aligned(b->seq_start_base, 4) || !aligned(b->kv_len_base, 4) || !aligned(b->page_table_base, 4))
    return fail(OPS_STRIDES_NOT_SUPPORT, "%s: the batch's arrays must be 4-byte aligned", op);
  if (m.npages && m.nkvh)
    for (int i = 0; i < 2; ++i) {
      if (!bases[i]) return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: null base pointer of the cache at launch", op);
      if (!aligned(bases[i], 16)) return fail(OPS_STRIDES_NOT_SUPPORT, "%s: the cache must be 16-byte aligned", op);
    }
  out->table = (const uint32_t *)b->page_table_base;
  out->start = (const uint32_t *)b->seq_start_base;
  out->len = (const uint32_t *)b->kv_len_base;
  out->table_ld = m.nseq > 1 ? b->page_table_layout.strides[0] / 4 : 0;
  out->nseq = (int)m.nseq;
  out->width = (int)m.width;
  out->nt = (int)nt;
  out->npages = (uint32_t)m.npages;
  out->max_seq = b->max_seq == 0 || b->max_seq > 0xfffffffeu ? 0xffffffffu : (uint32_t)b->max_seq;
  out->page_log2 = m.page_log2;
  out->status = status;
  return OPS_OK;
}

// Rows of 16-bit elements that are read and written 16 bytes at a time: dims in front of dh, unit inner stride.
inline int rows16_checks(const char *op, const char *what, const ops_layout *l, const void *base, bool any_sign) {
  const int last = (int)l->ndim - 1;
  bool empty = false;
  for (int d = 0; d <= last; ++d) {
    if (dyn(l->shape[d]) || dyn(l->strides[d])) return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: every shape and stride of %s must be static at launch", op, what);
    empty |= l->shape[d] == 0;
  }
  if (empty) return OPS_OK;
  if (l->strides[last] != 2) return fail(OPS_STRIDES_NOT_SUPPORT, "%s: last dim of %s must be contiguous", op, what);
  for (int d = 0; d < last; ++d)
    if (l->shape[d] > 1 && (l->strides[d] % 16 || (!any_sign && l->strides[d] <= 0) || l->strides[d] >= ((isz)1 << 40)))
      return fail(OPS_STRIDES_NOT_SUPPORT, "%s: strides of %s must be multiples of 16 bytes%s", op, what, any_sign ? "" : " and positive");
  if (!base) return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: null base pointer of %s at launch", op, what);
  if (!aligned(base, 16)) return fail(OPS_STRIDES_NOT_SUPPORT, "%s: %s must be 16-byte aligned", op, what);
  return OPS_OK;
}

// A handle that owns two status words on its device: what was wrong with a batch, and which bounded wait ran out.
struct PagedHandle {
  OpBase base;
  int *status;
  mutable std::atomic<unsigned> prepared{0};  // kernels whose shared memory has been reserved on the device
  std::atomic<unsigned long long> patience{100000};  // attention_paged's, ns: parts of a unit end within a few us of each other
};
int paged_create(PagedHandle *h, int device);
void paged_destroy(PagedHandle *h);
int paged_status(const PagedHandle *h);
int paged_status_reset(PagedHandle *h);

}  // namespace ops

#define OPS_DEFINE_PAGED_HANDLE(NAME)                                                                  \
  struct ops_##NAME {                                                                                  \
    ops::PagedHandle h;                                                                                \
  };                                                                                                   \
  OPS_API int ops_##NAME##_create(int device, ops_##NAME **out) {                                      \
    if (!out) return ops::fail(OPS_ARGS_NOT_SUPPORT, "null out pointer");                              \
    ops_##NAME *op = new (std::nothrow) ops_##NAME();                                                  \
    if (!op) return ops::fail(OPS_EXECUTION_FAILED, #NAME ": out of host memory");                     \
    int rc = ops::paged_create(&op->h, device);                                                        \
    if (rc != OPS_OK) {                                                                                \
      delete op;                                                                                       \
      return rc;                                                                                       \
    }                                                                                                  \
    *out = op;                                                                                         \
    return OPS_OK;                                                                                     \
  }                                                                                                    \
  OPS_API void ops_##NAME##_destroy(ops_##NAME *op) {                                                  \
    if (!op) return;                                                                                   \
    ops::paged_destroy(&op->h);                                                                        \
    delete op;                                                                                         \
  }                                                                                                    \
  OPS_API int ops_##NAME##_status(const ops_##NAME *op) { return op ? ops::paged_status(&op->h) : -1; } \
  OPS_API int ops_##NAME##_status_reset(ops_##NAME *op) {                                              \
    return op ? ops::paged_status_reset(&op->h) : ops::fail(OPS_ARGS_NOT_SUPPORT, "null handle");      \
  }
