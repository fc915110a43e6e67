// attention_paged.cu — attention of a batch of sequences' new tokens over their pages of a cache.
#include "attention_paged.h"

#include <algorithm>

#include "device_utils.cuh"

namespace ops {

// Clears the counters of the launch.  The kernel that uses them starts beside it and waits for it.
__global__ void __launch_bounds__(1024) attention_paged_clear_kernel(uint4 *counters, int n) {
  pdl_let_next_come();
  for (int i = threadIdx.x; i < n; i += 1024) counters[i] = make_uint4(0, 0, 0, 0);
}

// cuTensorMapEncodeTiled through the runtime's driver entry point
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return (EncodeTiledFn)p;
  }();
  return fn;
}

// A 4-d map of 16-bit elements, 64 of the innermost dim and `box1` x `box2` of the next two a box, 128-byte swizzle.
static bool ap_encode(CUtensorMap *map, bool bf16, const void *ptr, const usz (&dims)[4], const isz (&strides)[3], uint32_t box1, uint32_t box2) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[4], st[3];
  for (int i = 0; i < 4; ++i) d[i] = dims[i];
  for (int i = 0; i < 3; ++i) st[i] = dims[i + 1] > 1 ? (cuuint64_t)strides[i] : (cuuint64_t)(dims[0] * 2);  // never stepped over
  cuuint32_t box[4] = {64, box1, box2, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(ptr), d, st, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool ap_encode_cache(const PagedAttnArgs &a, bool bf16, const PagedLineArgs &l, CUtensorMap *k, CUtensorMap *v) {
  const usz dims[4] = {(usz)a.dh, (usz)1 << a.batch.page_log2, (usz)l.line.nkvh, a.batch.npages};
  const isz ks[3] = {a.kp_s, a.kp_h, a.kp_p}, vs[3] = {a.vp_s, a.vp_h, a.vp_p};
  return ap_encode(k, bf16, a.k, dims, ks, 1u << l.box_log2, 1) && ap_encode(v, bf16, a.v, dims, vs, 1u << l.box_log2, 1);
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

OPS_API int ops_attention_paged_set_patience(ops_attention_paged *op, uint64_t nanoseconds) {
  if (!op) return fail(OPS_ARGS_NOT_SUPPORT, "null handle");
  if (nanoseconds > 1000000000u) return fail(OPS_ARGS_NOT_SUPPORT, "attention_paged: a patience of %llu ns, 1 s at most expected", (unsigned long long)nanoseconds);
  op->h.patience.store(nanoseconds, std::memory_order_relaxed);
  return OPS_OK;
}

namespace ops {

// The two lines of a launch and the scratch they want.  Where max_seq says that there are no tiles, the launch is of the kernel
// without them.
struct PagedAttnPlan : PagedLines {
  int part_dh;
  usz few_arrived, tile_arrived, few_parts, tile_parts;  // bytes
  usz bytes() const { return few_arrived + tile_arrived + few_parts + tile_parts + 256; }
};

static usz up256(usz n) { return (n + 255) / 256 * 256; }

static PagedAttnPlan attention_paged_plan(const OpBase &base, usz nh, usz nkvh, usz dh, bool causal, uint32_t max_seq, usz nt, usz nseq, usz slots) {
  PagedAttnPlan p;
  static_cast<PagedLines &>(p) = paged_lines(base.sm_count, nh, nkvh, causal, max_seq, nt, nseq, slots);
  p.part_dh = dh <= 64 ? 64 : 128;
  p.few_arrived = up256((usz)AP_LEVELS * p.few.ctas * 8 * sizeof(uint32_t));
  p.few_parts = up256(3 * (usz)p.few.ctas * p.few_rows * (p.part_dh + 2) * sizeof(float));
  p.tile_arrived = up256((usz)AP_LEVELS * p.tile.ctas * 8 * sizeof(uint32_t));
  p.tile_parts = up256(2 * (usz)p.tile.ctas * AP_TILE_ROWS * (p.part_dh + 2) * sizeof(float));
  return p;
}

}  // namespace ops

OPS_API int ops_attention_paged_scheme(ops_attention_paged *op, const ops_attention_paged_args *args, size_t max_ws, size_t *ws_out) {
  PagedAttnMeta m;
  OPS_TRY(attention_paged_meta(args, &m));
  if (ws_out) {
    *ws_out = 0;
    if (!dyn(m.nh) && !dyn(m.paged.nkvh) && !dyn(m.dh) && m.nh && m.paged.nkvh) {
      OpBase none{0, 148};
      const uint32_t max_seq = args->batch.max_seq == 0 || args->batch.max_seq > 0xfffffffeu ? 0xffffffffu : (uint32_t)args->batch.max_seq;
      const usz need = attention_paged_plan(op ? op->h.base : none, m.nh, m.paged.nkvh, m.dh, args->mask == OPS_MASK_CAUSAL, max_seq, 1, 1, 1).bytes();
      *ws_out = need <= max_ws ? need : 0;
    }
  }
  return OPS_OK;
}

OPS_API int ops_attention_paged_launch(const ops_attention_paged *op, const ops_attention_paged_args *a, void *ws, size_t ws_len, void *stream) {
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
  if (m.paged.npages == 0) return fail(OPS_SHAPE_NOT_SUPPORT, "attention_paged: a cache without pages");
  const OpBase base = op ? op->h.base : OpBase{0, 148};
  const PagedAttnPlan plan = attention_paged_plan(base, m.nh, m.paged.nkvh, m.dh, a->mask == OPS_MASK_CAUSAL, g.batch.max_seq, m.nt, m.paged.nseq,
                                                m.paged.width * m.paged.page);
  if (!plan.fit) return fail(OPS_SHAPE_NOT_SUPPORT, "attention_paged: more than some 2^29 units of a sequence, a kv head and its query rows");
  if (!op) return fail(OPS_ARGS_NOT_SUPPORT, "null handle");
  if (!ws || ws_len < plan.bytes()) return need_workspace(plan.bytes());
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
  g.dh = (int)m.dh;
  g.scale_log2 = a->scale * 1.4426950408889634f;
  DeviceGuard guard(base.device);
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf16 = m.dt == OPS_DT_BF16;
  char *at = (char *)(((uintptr_t)ws + 255) / 256 * 256);
  g.patience = op->h.patience.load(std::memory_order_relaxed);
  g.odd_scale = !(g.scale_log2 > 0.f);
  g.per_tile = AP_TILE_ROWS / 2 / (int)(m.nh / m.paged.nkvh);
  g.few.line = plan.few;
  g.few.box_log2 = std::min(m.paged.page_log2, AP_FEW_BLOCK_LOG2);
  g.few.arrived = (uint32_t *)at;
  g.few.parts = (float *)(at + plan.few_arrived + plan.tile_arrived);
  g.few.parts_ml = (float2 *)(g.few.parts + 3 * (usz)plan.few.ctas * plan.few_rows * plan.part_dh);
  g.tile.line = plan.tile;
  g.tile.box_log2 = std::min(m.paged.page_log2, 6);
  g.tile.arrived = (uint32_t *)(at + plan.few_arrived);
  g.tile.parts = (float *)(at + plan.few_arrived + plan.tile_arrived + plan.few_parts);
  g.tile.parts_ml = (float2 *)(g.tile.parts + 2 * (usz)plan.tile.ctas * AP_TILE_ROWS * plan.part_dh);
  if (plan.few.ctas && plan.tile.ctas)
    for (int k = 0; k < AP_SHARES; ++k) {
      const int share = paged_share(plan.few.ctas, k);
      g.few.by_ctas[k] = paged_div_by((uint32_t)share);
      g.tile.by_ctas[k] = paged_div_by((uint32_t)std::max(1, plan.tile.ctas - share));
    }
  PagedAttnMaps maps;
  memset(&maps, 0, sizeof(maps));
  bool made = true;
  if (plan.few.ctas) made = ap_encode_cache(g, bf16, g.few, &maps.few_k, &maps.few_v);
  if (plan.tile.ctas) {
    const usz q_dims[4] = {m.dh, (usz)plan.tile.group, m.nt, m.paged.nkvh};
    const isz q_st[3] = {g.q_h, g.q_t, g.q_h * plan.tile.group};
    made = made && ap_encode(&maps.tile_q, bf16, g.q, q_dims, q_st, (uint32_t)plan.tile.group, (uint32_t)g.per_tile) && ap_encode_cache(g, bf16, g.tile, &maps.tile_k, &maps.tile_v);
  }
  if (!made) return fail(OPS_EXECUTION_FAILED, "attention_paged: cuTensorMapEncodeTiled failed");
  attention_paged_clear_kernel<<<1, 1024, 0, s>>>((uint4 *)at, (int)((plan.few_arrived + plan.tile_arrived) / 16));
  OPS_TRY(check_launch("attention_paged(clear)"));
  OPS_TRY((bf16 ? attention_paged_run_bf16 : attention_paged_run_f16)(maps, g, plan.few_rows, plan.tile.ctas > 0, op->h.prepared, s));
  return OPS_OK;
}
