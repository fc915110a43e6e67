// attention_paged.cu — attention of a batch of sequences' new tokens over their pages of a cache.
#include "attention_paged.h"

#include <algorithm>

#include "device_utils.cuh"

namespace ops {

// Joins the parts of the units that several CTAs share:
//   o = sum_d 2^(m_d - M) O_d / sum_d 2^(m_d - M) l_d,  M = max_d m_d, parts in the order of their keys.
// Block (c, y) takes rows [16 y, 16 y + 16) of the unit whose first blocks CTA c had.  With fewer rows a row's parts are dealt to
// several warps, which meet in shared memory; a lane holds 4 columns.
constexpr int JOIN_WARPS = 16, JOIN_ROWS = 16;

template <bool BF>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attention_paged_join_kernel(const __grid_constant__ PagedAttnArgs few, const __grid_constant__ PagedAttnArgs tile,
                                                                              int few_rows, int tile_rows, int part_dh) {
  pdl_wait_for_front();
  const bool on_tile = (int)blockIdx.x >= few.line.ctas;
  const PagedAttnArgs &a = on_tile ? tile : few;
  const int first = on_tile ? blockIdx.x - few.line.ctas : blockIdx.x;
  const PagedJoin j = a.joins[first];
  const int group = a.line.group, rows = j.ctas ? j.tokens * group : 0;
  const int row0 = blockIdx.y * JOIN_ROWS, here = min(JOIN_ROWS, rows - row0);
  if (here <= 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = JOIN_WARPS / here;  // warps per row
  const int mine = warp / share, part = warp - mine * share;
  const int r = row0 + mine;
  // where the row lies in a parked unit: tiles of 128 rows, whole tokens each
  const int tok = r / group, gi = r - tok * group;
  const int per_tile = on_tile ? 128 / group : JOIN_ROWS, t = tok / per_tile;
  const int parked = t * 128 + (tok - t * per_tile) * group + gi;
  const long long ld = part_dh + AP_PAD, unit = (long long)(on_tile ? tile_rows : few_rows) * ld;
  __shared__ float meet[JOIN_WARPS][AP_MAX_DH + 2];
  __shared__ short slot_s[AP_MAX_CTAS];  // of the part of the d-th CTA behind the first; -1: the cut left it none
  for (int d = threadIdx.x; d < j.ctas; d += JOIN_WARPS * 32) {
    PagedUnit u;
    u.head = u.tile = 0;
    u.begin = j.begin;
    u.cost = j.cost;
    const int c = first + d;
    const int lo = paged_block(a.line, u, j.blocks, paged_cut(j.total, j.active, c));
    const int hi = paged_block(a.line, u, j.blocks, c + 1 < j.active ? paged_cut(j.total, j.active, c + 1) : j.total);
    slot_s[d] = (short)(lo >= hi ? -1 : c * 2 + (lo > 0 ? 0 : 1));
  }
  __syncthreads();
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine < here) {
    constexpr int DEEP = 4;
    for (int d0 = part; d0 < j.ctas; d0 += share * DEEP) {
      float4 v[DEEP];
      float2 ml[DEEP];
#pragma unroll
      for (int e = 0; e < DEEP; ++e) {
        const int d = d0 + e * share;
        v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        ml[e] = make_float2(-INFINITY, 0.f);
        const int slot = d < j.ctas ? slot_s[d] : -1;
        if (slot >= 0) {
          const float *from = a.parts + slot * unit + parked * ld;
          ml[e] = __ldcg(reinterpret_cast<const float2 *>(from + part_dh));
          if (lane * 4 < a.dh) v[e] = __ldcg(reinterpret_cast<const float4 *>(from + lane * 4));
        }
      }
#pragma unroll
      for (int e = 0; e < DEEP; ++e) {
        if (ml[e].x == -INFINITY) continue;  // a part in which the row sees nothing may have left its o unwritten
        const float top = fmaxf(m, ml[e].x);
        const float at = top == -INFINITY ? 0.f : top;
        const float wa = ap_ex2(m - at), wb = ap_ex2(ml[e].x - at);
        l = l * wa + ml[e].y * wb;
        acc.x = acc.x * wa + v[e].x * wb;
        acc.y = acc.y * wa + v[e].y * wb;
        acc.z = acc.z * wa + v[e].z * wb;
        acc.w = acc.w * wa + v[e].w * wb;
        m = top;
      }
    }
    if (part > 0) {
      *reinterpret_cast<float2 *>(&meet[warp][lane * 4]) = make_float2(acc.x, acc.y);
      *reinterpret_cast<float2 *>(&meet[warp][lane * 4 + 2]) = make_float2(acc.z, acc.w);
      if (lane == 0) {
        meet[warp][AP_MAX_DH] = m;
        meet[warp][AP_MAX_DH + 1] = l;
      }
    }
  }
  __syncthreads();
  if (mine >= here || part > 0) return;
  for (int w = warp + 1; w < warp + share; ++w) {
    const float mw = meet[w][AP_MAX_DH], top = fmaxf(m, mw);
    const float at = top == -INFINITY ? 0.f : top;
    const float wa = ap_ex2(m - at), wb = ap_ex2(mw - at);
    l = l * wa + meet[w][AP_MAX_DH + 1] * wb;
    acc.x = acc.x * wa + meet[w][lane * 4] * wb;
    acc.y = acc.y * wa + meet[w][lane * 4 + 1] * wb;
    acc.z = acc.z * wa + meet[w][lane * 4 + 2] * wb;
    acc.w = acc.w * wa + meet[w][lane * 4 + 3] * wb;
    m = top;
  }
  if (lane * 4 >= a.dh) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  char *to = a.o + (long long)(j.row + tok) * a.o_t + (long long)(j.head * group + gi) * a.o_h + lane * 8;
  *reinterpret_cast<uint2 *>(to) = make_uint2(ap_pack<BF>(acc.x * inv, acc.y * inv), ap_pack<BF>(acc.z * inv, acc.w * inv));
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

namespace ops {

// Which kernels a launch takes, and the scratch they want.  A sequence goes to the few-rows kernel when its new tokens times the
// query heads of a kv head fit its rows; sequences with more go to the tile kernel.  What no sequence can need by max_seq is left
// out of the launch.
struct PagedAttnPlan {
  PagedLine few, tile;  // ctas == 0: not launched
  int few_rows, part_dh;
  usz few_joins, few_parts, tile_joins, tile_parts;  // bytes
  usz bytes() const { return few_joins + few_parts + tile_joins + tile_parts + 256; }
};

static usz up256(usz n) { return (n + 255) / 256 * 256; }

static PagedAttnPlan attention_paged_plan(const OpBase &base, usz nh, usz nkvh, usz dh, bool causal, uint32_t max_seq) {
  PagedAttnPlan p;
  memset(&p, 0, sizeof(p));
  const usz group = nh / nkvh, most = max_seq == 0xffffffffu ? 0xffffffffull : (usz)max_seq * group;
  // 16 rows cost the kernel half its CTAs; 8 are enough for one token of up to 8 heads
  p.few_rows = group <= 8 && !(most > 8 && most <= 16) ? 8 : 16;
  p.part_dh = dh <= 64 ? 64 : 128;
  PagedLine l;
  memset(&l, 0, sizeof(l));
  l.nkvh = (int)nkvh;
  l.group = (int)group;
  l.causal = causal;
  l.max_seq = max_seq > 0x7fffffffu ? 0x7fffffff : (int)max_seq;
  p.few = p.tile = l;
  if (group <= (usz)p.few_rows) {
    p.few.rows_lo = 1;
    p.few.rows_hi = p.few_rows;
    p.few.tokens = p.few_rows;
    p.few.block = AP_FEW_BLOCK;
    p.few.overhead = 128;
    p.few.min_share = 256;
    p.few.ctas = std::min(attention_paged_few_ctas(base, p.few_rows), AP_MAX_CTAS);
    p.few_joins = up256(sizeof(PagedJoin) * (usz)p.few.ctas);
    p.few_parts = up256(2 * (usz)p.few.ctas * p.few_rows * (p.part_dh + AP_PAD) * sizeof(float));
    p.tile.rows_lo = p.few_rows + 1;
  } else {
    p.tile.rows_lo = 1;
  }
  if (most >= (usz)p.tile.rows_lo) {
    p.tile.rows_hi = 0x7fffffff;
    p.tile.tokens = AP_TILE_ROWS / 2 / (int)group * 2;
    p.tile.block = AP_TILE_BLOCK;
    p.tile.overhead = 256;
    p.tile.min_share = 512;
    p.tile.ctas = std::min(base.sm_count, AP_MAX_CTAS);
    p.tile_joins = up256(sizeof(PagedJoin) * (usz)p.tile.ctas);
    p.tile_parts = up256(2 * (usz)p.tile.ctas * AP_TILE_ROWS * (p.part_dh + AP_PAD) * sizeof(float));
  }
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
      const usz need = attention_paged_plan(op ? op->h.base : none, m.nh, m.paged.nkvh, m.dh, args->mask == OPS_MASK_CAUSAL, max_seq).bytes();
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
  if (!op) return fail(OPS_ARGS_NOT_SUPPORT, "null handle");
  const OpBase &base = op->h.base;
  const PagedAttnPlan plan = attention_paged_plan(base, m.nh, m.paged.nkvh, m.dh, a->mask == OPS_MASK_CAUSAL, g.batch.max_seq);
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
  PagedAttnArgs few = g, tile = g;
  few.line = plan.few;
  few.joins = (PagedJoin *)at;
  few.parts = (float *)(at + plan.few_joins);
  tile.line = plan.tile;
  tile.joins = (PagedJoin *)(at + plan.few_joins + plan.few_parts);
  tile.parts = (float *)(at + plan.few_joins + plan.few_parts + plan.tile_joins);
  if (plan.few.ctas) OPS_TRY(attention_paged_few(few, plan.few_rows, bf16, s));
  if (plan.tile.ctas) OPS_TRY(attention_paged_tile(tile, bf16, s));
  if (plan.few.ctas + plan.tile.ctas) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(plan.few.ctas + plan.tile.ctas), plan.tile.ctas ? AP_TILE_ROWS / JOIN_ROWS : 1);
    cfg.blockDim = dim3(JOIN_WARPS * 32);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = bf16 ? cudaLaunchKernelEx(&cfg, attention_paged_join_kernel<true>, few, tile, plan.few_rows, AP_TILE_ROWS, plan.part_dh)
                         : cudaLaunchKernelEx(&cfg, attention_paged_join_kernel<false>, few, tile, plan.few_rows, AP_TILE_ROWS, plan.part_dh);
    if (e != cudaSuccess) return fail(OPS_EXECUTION_FAILED, "attention_paged: launch of the joining kernel failed: %s", cudaGetErrorString(e));
  }
  return OPS_OK;
}
