// attention_paged.cu — attention of a batch of sequences' new tokens over their pages of a cache.
#include "device_utils.cuh"
#include "paged.h"

namespace ops {

constexpr int AP_MAX_DH = 128;
constexpr int AP_MAX_GROUP = 128;

struct PagedAttnArgs {
  const char *q, *k, *v;
  char *o;
  long long q_h, q_t, o_h, o_t;                  // byte strides: head, token
  long long kp_p, kp_h, kp_s, vp_p, vp_h, vp_s;  // byte strides: page, head, slot
  int nh, group, dh, causal;
  float scale_log2;  // scale * log2(e): the softmax runs in powers of two
  PagedBatch batch;
};

// One warp per (token, head).
template <class E>
__global__ void __launch_bounds__(128) attention_paged_rows_kernel(const __grid_constant__ PagedAttnArgs a) {
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int tok = (int)(item / a.nh), head = (int)(item - (long long)tok * a.nh), kvh = head / a.group;
  if (tok >= a.batch.nt) return;
  const int i = paged_find(a.batch, (uint32_t)tok);
  if (i < 0) return;
  const PagedSeq s = paged_seq(a.batch, i, lane == 0);
  if (tok - s.row >= s.n || (uint32_t)s.n > a.batch.max_seq) return;
  const int seen = a.causal ? max(0, s.len - s.n + (tok - s.row) + 1) : s.len;
  const E *q = reinterpret_cast<const E *>(a.q + (long long)tok * a.q_t + (long long)head * a.q_h);
  __shared__ float q_s[4][AP_MAX_DH];
  float *qw = q_s[threadIdx.x >> 5];
  for (int d = lane; d < a.dh; d += 32) qw[d] = to_f32(q[d]);
  __syncwarp();
  const uint32_t *table = a.batch.table + (long long)i * a.batch.table_ld;
  const int mask = (1 << a.batch.page_log2) - 1;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < seen; k0 += 32) {
    const int key = k0 + lane;
    uint32_t page = 0xffffffffu;
    float x = -INFINITY;
    if (key < seen) {
      page = table[key >> a.batch.page_log2];
      x = 0.f;
      if (page < a.batch.npages) {
        const E *k = reinterpret_cast<const E *>(a.k + (long long)page * a.kp_p + (long long)kvh * a.kp_h + (long long)(key & mask) * a.kp_s);
        for (int d = 0; d < a.dh; d += 8) {
          Vec8<E> kv;
          kv.u = ld_global_16(k + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) x = fmaf(qw[d + e], to_f32(kv.h[e]), x);
        }
      } else {
        atomicCAS(a.batch.status, 0, OPS_PAGED_BAD_PAGE);
      }
      x *= a.scale_log2;
    }
    const float m_new = fmaxf(m, warp_max(x));
    const float at = m_new == -INFINITY ? 0.f : m_new;
    const float p = exp2f(x - at), alpha = exp2f(m - at);
    l = fmaf(l, alpha, warp_sum(p));
    m = m_new;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= alpha;
    for (int j = 0; j < min(32, seen - k0); ++j) {
      const uint32_t pg = __shfl_sync(0xffffffffu, page, j);
      const float pj = __shfl_sync(0xffffffffu, p, j);
      if (pg < a.batch.npages && lane * 4 < a.dh) {
        const E *v = reinterpret_cast<const E *>(a.v + (long long)pg * a.vp_p + (long long)kvh * a.vp_h + (long long)((k0 + j) & mask) * a.vp_s) + lane * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(pj, to_f32(v[e]), o[e]);
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  E *out = reinterpret_cast<E *>(a.o + (long long)tok * a.o_t + (long long)head * a.o_h) + lane * 4;
  if (lane * 4 < a.dh)
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = from_f32<E>(o[e] * inv);
}

struct PagedAttnMeta {
  uint32_t dt;
  usz nt, nh, dh;
  PagedMeta paged;
};

static int attention_paged_meta(const ops_attention_paged_args *a, PagedAttnMeta *m) {
  if (a->q_layout.ndim != 3) return fail(OPS_RANK_NOT_SUPPORT, "q.ndim = %u, 3 expected", a->q_layout.ndim);
  if (a->o_layout.ndim != 3) return fail(OPS_RANK_NOT_SUPPORT, "o.ndim = %u, 3 expected", a->o_layout.ndim);
  OPS_TRY(paged_meta(&a->batch, &a->k_pages_layout, &a->v_pages_layout, &m->paged));
  m->dt = a->q_layout.dt;
  if (m->dt != OPS_DT_F16 && m->dt != OPS_DT_BF16) return fail(OPS_TYPE_NOT_SUPPORT, "attention_paged: f16 or bf16 expected");
  if (a->o_layout.dt != m->dt || a->k_pages_layout.dt != m->dt || a->v_pages_layout.dt != m->dt)
    return fail(OPS_TYPE_MISMATCH, "element types of q, o and the cache differ");
  if (a->mask != OPS_MASK_NONE && a->mask != OPS_MASK_CAUSAL) return fail(OPS_ARGS_NOT_SUPPORT, "attention_paged: unknown mask %u", a->mask);
  const usz nhs[2] = {a->q_layout.shape[0], a->o_layout.shape[0]};
  const usz nts[2] = {a->q_layout.shape[1], a->o_layout.shape[1]};
  const usz dhs[3] = {a->q_layout.shape[2], a->o_layout.shape[2], m->paged.dh};
  if (!merge_dims(nhs, 2, &m->nh)) return fail(OPS_SHAPE_MISMATCH, "nh of q and o differ");
  if (!merge_dims(nts, 2, &m->nt)) return fail(OPS_SHAPE_MISMATCH, "nt of q and o differ");
  if (!merge_dims(dhs, 3, &m->dh)) return fail(OPS_SHAPE_MISMATCH, "dh of q, o and the cache differ");
  if (!dyn(m->nh) && !dyn(m->paged.nkvh)) {
    if (m->paged.nkvh == 0 ? m->nh != 0 : m->nh % m->paged.nkvh != 0) return fail(OPS_SHAPE_MISMATCH, "attention_paged: nh must be a multiple of nkvh");
    if (m->paged.nkvh && m->nh / m->paged.nkvh > (usz)AP_MAX_GROUP) return fail(OPS_SHAPE_NOT_SUPPORT, "attention_paged: more than %d query heads per kv head", AP_MAX_GROUP);
  }
  if (!dyn(m->dh) && (m->dh % 8 || m->dh > (usz)AP_MAX_DH)) return fail(OPS_SHAPE_NOT_SUPPORT, "attention_paged: dh = %zu, a multiple of 8 up to %d expected", m->dh, AP_MAX_DH);
  if (!dyn(m->nh) && m->nh > 0xffffu) return fail(OPS_SHAPE_NOT_SUPPORT, "attention_paged: too many heads");
  return OPS_OK;
}

}  // namespace ops

using namespace ops;

OPS_DEFINE_PAGED_HANDLE(attention_paged)

OPS_API int ops_attention_paged_scheme(ops_attention_paged *op, const ops_attention_paged_args *args, size_t max_ws, size_t *ws_out) {
  (void)op;
  (void)max_ws;
  PagedAttnMeta m;
  OPS_TRY(attention_paged_meta(args, &m));
  if (ws_out) *ws_out = 0;
  return OPS_OK;
}

OPS_API int ops_attention_paged_launch(const ops_attention_paged *op, const ops_attention_paged_args *a, void *ws, size_t ws_len, void *stream) {
  (void)ws;
  (void)ws_len;
  static const char *name = "attention_paged";
  PagedAttnMeta m;
  OPS_TRY(attention_paged_meta(a, &m));
  if (dyn(a->scale)) return fail(OPS_DYNAMIC_NOT_SUPPORT, "attention_paged: scale must be static at launch");
  PagedAttnArgs g;
  memset(&g, 0, sizeof(g));
  OPS_TRY(rows16_checks(name, "q", &a->q_layout, a->q_base, false));
  OPS_TRY(rows16_checks(name, "o", &a->o_layout, a->o_base, false));
  OPS_TRY(paged_launch_checks(name, &a->batch, &a->k_pages_layout, a->k_pages_base, &a->v_pages_layout, a->v_pages_base, m.paged, m.nt,
                              op ? op->h.status : nullptr, &g.batch));
  if (m.nt == 0 || m.nh == 0 || m.dh == 0 || m.paged.nseq == 0) return OPS_OK;
  if (!op) return fail(OPS_ARGS_NOT_SUPPORT, "null handle");
  g.q = (const char *)a->q_base;
  g.q_h = a->q_layout.strides[0];
  g.q_t = a->q_layout.strides[1];
  g.o = (char *)a->o_base;
  g.o_h = a->o_layout.strides[0];
  g.o_t = a->o_layout.strides[1];
  g.k = (const char *)a->k_pages_base;
  g.v = (const char *)a->v_pages_base;
  const isz *sk = a->k_pages_layout.strides, *sv = a->v_pages_layout.strides;
  g.kp_p = sk[0];
  g.kp_h = sk[1];
  g.kp_s = sk[2];
  g.vp_p = sv[0];
  g.vp_h = sv[1];
  g.vp_s = sv[2];
  g.nh = (int)m.nh;
  g.group = (int)(m.nh / m.paged.nkvh);
  g.dh = (int)m.dh;
  g.causal = a->mask == OPS_MASK_CAUSAL;
  g.scale_log2 = a->scale * 1.4426950408889634f;
  DeviceGuard guard(op->h.base.device);
  const unsigned long long items = (unsigned long long)m.nt * m.nh;
  if (items > 0x7fffffffull) return fail(OPS_SHAPE_NOT_SUPPORT, "attention_paged: shape too large");
  const unsigned grid = (unsigned)((items + 3) / 4);
  if (m.dt == OPS_DT_BF16) attention_paged_rows_kernel<__nv_bfloat16><<<grid, 128, 0, (cudaStream_t)stream>>>(g);
  else attention_paged_rows_kernel<__half><<<grid, 128, 0, (cudaStream_t)stream>>>(g);
  return check_launch(name);
}
