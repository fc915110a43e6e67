// attention_paged.cu — attention of a batch of sequences' new tokens over their pages of a cache.
#include "attention_paged.h"

#include <algorithm>

#include "device_utils.cuh"

namespace ops {

// Joins the parts of the units that several CTAs share:
//   o = sum_d 2^(m_d - M) O_d / sum_d 2^(m_d - M) l_d,  M = max_d m_d, parts in the order of their keys.
// An item is 16 rows of a unit.  How many units there are, and of how many rows and parts, only the records tell (one long
// sequence: few units of a hundred parts; a prompt: a unit per CTA, of two), so every block counts the items of all records and
// the blocks deal them out among themselves.  With fewer than 16 rows a row's parts go to several warps, which meet in shared
// memory; a lane holds 4 columns.
constexpr int JOIN_WARPS = 16, JOIN_THREADS = JOIN_WARPS * 32, JOIN_ROWS = 16;
constexpr int JOIN_BLOCKS_PER_SM = 2;

template <bool BF>
__global__ void __launch_bounds__(JOIN_THREADS, JOIN_BLOCKS_PER_SM)
    attention_paged_join_kernel(const __grid_constant__ PagedAttnArgs few, const __grid_constant__ PagedAttnArgs tile, int few_rows, int part_dh) {
  __shared__ int first_item[2 * AP_MAX_CTAS];  // of every record
  __shared__ PagedJoin joins[2 * AP_MAX_CTAS];
  __shared__ int warp_items[JOIN_WARPS];
  __shared__ __align__(16) float meet[JOIN_WARPS][AP_MAX_DH + AP_PAD];  // o, m, l; 16-byte rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int records = few.line.ctas + tile.line.ctas, group = few.line.group;
  pdl_wait_for_front();
  // items in front of every record's: a prefix sum over rounds of a record per thread
  int items = 0;
  for (int j0 = 0; j0 < records; j0 += JOIN_THREADS) {
    const int j = j0 + threadIdx.x;
    int mine = 0;
    if (j < records) {
      const PagedJoin rec = j < few.line.ctas ? few.joins[j] : tile.joins[j - few.line.ctas];
      joins[j] = rec;
      if (rec.ctas) mine = (rec.tokens * group + JOIN_ROWS - 1) / JOIN_ROWS;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) warp_items[warp] = upto;
    __syncthreads();
    int sum = warp_items[lane & (JOIN_WARPS - 1)];  // of all warps, by every warp for itself
#pragma unroll
    for (int o = 1; o < JOIN_WARPS; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if ((lane & (JOIN_WARPS - 1)) >= o) sum += x;
    }
    const int front = warp == 0 ? 0 : __shfl_sync(0xffffffffu, sum, warp - 1);
    if (j < records) first_item[j] = items + front + upto - mine;
    items += __shfl_sync(0xffffffffu, sum, JOIN_WARPS - 1);
    __syncthreads();
  }

  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    int lo = 0, hi = records;  // the last record whose first item is at or before this one has it
#pragma unroll 1
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first_item[mid] <= item) lo = mid;
      else hi = mid;
    }
    const bool on_tile = lo >= few.line.ctas;
    const PagedAttnArgs &a = on_tile ? tile : few;
    const PagedJoin &j = joins[lo];
    const int first = on_tile ? lo - few.line.ctas : lo;
    const int row0 = (item - first_item[lo]) * JOIN_ROWS, here = min(JOIN_ROWS, j.tokens * group - row0);
    const int share = here > 8 ? 1 : here > 5 ? 2 : here > 4 ? 3 : here > 3 ? 4 : here > 2 ? 5 : here > 1 ? 8 : 16;  // JOIN_WARPS / here warps per row
    const int own = paged_guess((float)warp + 0.5f, (float)share), part = warp - own * share;  // warp / share
    const int r = row0 + own;
    // where the row lies in a parked unit: tiles of 128 rows, whole tokens each
    const int tok = paged_div(r, few.line.by_group), gi = r - tok * group;
    const int per_tile = on_tile ? tile.line.tokens / 2 : JOIN_ROWS, t = tok >= per_tile;
    const int parked = t * (AP_TILE_ROWS / 2) + (tok - t * per_tile) * group + gi;
    const long long ld = part_dh + AP_PAD, unit = (long long)(on_tile ? AP_TILE_ROWS : few_rows) * ld;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (own < here) {
      constexpr int DEEP = 4;
      for (int d0 = part; d0 < j.ctas; d0 += share * DEEP) {
        float4 v[DEEP];
        float2 ml[DEEP];
#pragma unroll
        for (int e = 0; e < DEEP; ++e) {
          const int d = d0 + e * share;
          v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
          ml[e] = make_float2(-INFINITY, 0.f);
          // the first has the unit's beginning in its second slot; a cut may have left one of the others none
          const int slot = d >= j.ctas ? -1 : d == 0 ? first * 2 + 1 : joins[lo + d].front ? (first + d) * 2 : -1;
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
          const float wa = ap_ex2(m - top), wb = ap_ex2(ml[e].x - top);
          l = l * wa + ml[e].y * wb;
          acc.x = acc.x * wa + v[e].x * wb;
          acc.y = acc.y * wa + v[e].y * wb;
          acc.z = acc.z * wa + v[e].z * wb;
          acc.w = acc.w * wa + v[e].w * wb;
          m = top;
        }
      }
      if (part > 0) {
        *reinterpret_cast<float4 *>(&meet[warp][lane * 4]) = acc;
        if (lane == 0) {
          meet[warp][AP_MAX_DH] = m;
          meet[warp][AP_MAX_DH + 1] = l;
        }
      }
    }
    __syncthreads();
    if (own < here && part == 0) {
      for (int w = warp + 1; w < warp + share; ++w) {
        const float mw = meet[w][AP_MAX_DH], top = fmaxf(m, mw);
        if (mw == -INFINITY) continue;
        const float wa = ap_ex2(m - top), wb = ap_ex2(mw - top);
        l = l * wa + meet[w][AP_MAX_DH + 1] * wb;
        const float4 v = *reinterpret_cast<const float4 *>(&meet[w][lane * 4]);
        acc.x = acc.x * wa + v.x * wb;
        acc.y = acc.y * wa + v.y * wb;
        acc.z = acc.z * wa + v.z * wb;
        acc.w = acc.w * wa + v.w * wb;
        m = top;
      }
      if (lane * 4 < a.dh) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        char *to = a.o + (long long)(j.row + tok) * a.o_t + (long long)(j.head * group + gi) * a.o_h + lane * 8;
        *reinterpret_cast<uint2 *>(to) = make_uint2(ap_pack<BF>(acc.x * inv, acc.y * inv), ap_pack<BF>(acc.z * inv, acc.w * inv));
      }
    }
    __syncthreads();  // meet is free again
  }
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

bool ap_encode(CUtensorMap *map, bool bf16, const void *ptr, const usz (&dims)[4], const isz (&strides)[3], uint32_t box1, uint32_t box2) {
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

int attention_paged_maps(const PagedAttnArgs &a, bool bf16, uint32_t rows, CUtensorMap *k, CUtensorMap *v) {
  const usz dims[4] = {(usz)a.dh, (usz)1 << a.batch.page_log2, (usz)a.line.nkvh, a.batch.npages};
  const isz ks[3] = {a.kp_s, a.kp_h, a.kp_p}, vs[3] = {a.vp_s, a.vp_h, a.vp_p};
  if (!ap_encode(k, bf16, a.k, dims, ks, rows, 1) || !ap_encode(v, bf16, a.v, dims, vs, rows, 1))
    return fail(OPS_EXECUTION_FAILED, "attention_paged: cuTensorMapEncodeTiled failed");
  return OPS_OK;
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

// The least shift with which a line cannot pass 31 bits: units, at most all rows in tiles and one more per sequence, of at most
// all slots and rows.  `overhead`, `min_share`: keys.
static void line_scale(PagedLine *l, usz nt, usz nseq, usz slots, int overhead, int min_share) {
  const double units = ((double)(nt / (usz)l->tokens) + (double)nseq) * l->nkvh, keys = (double)slots + (double)nt + l->tokens + overhead;
  l->shift = 0;
  while (l->shift < 30 && units * (std::ldexp(keys, -l->shift) + 4.0) > 2147483647.0) ++l->shift;
  l->overhead = std::max(1, overhead >> l->shift);
  l->min_share = std::max(1, min_share >> l->shift);  // a power of two
  l->min_share_log2 = 0;
  while ((1 << l->min_share_log2) < l->min_share) ++l->min_share_log2;
  l->by_tokens = paged_div_by((uint32_t)l->tokens);
  l->by_ctas = paged_div_by((uint32_t)l->ctas);
}

static PagedAttnPlan attention_paged_plan(const OpBase &base, usz nh, usz nkvh, usz dh, bool causal, uint32_t max_seq, usz nt, usz nseq, usz slots) {
  PagedAttnPlan p;
  memset(&p, 0, sizeof(p));
  const usz group = nh / nkvh, most = max_seq == 0xffffffffu ? 0xffffffffull : (usz)max_seq * group;
  // 16 rows cost the kernel a third of its ring; 8 are enough for one token of up to 8 heads
  p.few_rows = group <= 8 && !(most > 8 && most <= 16) ? 8 : 16;
  p.part_dh = dh <= 64 ? 64 : 128;
  PagedLine l;
  memset(&l, 0, sizeof(l));
  l.nkvh = (int)nkvh;
  l.group = (int)group;
  l.by_group = paged_div_by((uint32_t)group);
  l.causal = causal;
  l.max_seq = max_seq > 0x7fffffffu ? 0x7fffffff : (int)max_seq;
  p.few = p.tile = l;
  if (group <= (usz)p.few_rows) {
    p.few.rows_lo = 1;
    p.few.rows_hi = p.few_rows;
    p.few.tokens = p.few_rows;
    p.few.block_log2 = AP_FEW_BLOCK_LOG2;
    p.few.ctas = std::min(attention_paged_few_ctas(base), AP_MAX_CTAS);
    line_scale(&p.few, nt, nseq, slots, 128, 128);
    p.few_joins = up256(sizeof(PagedJoin) * (usz)p.few.ctas);
    p.few_parts = up256(2 * (usz)p.few.ctas * p.few_rows * (p.part_dh + AP_PAD) * sizeof(float));
    p.tile.rows_lo = p.few_rows + 1;
  } else {
    p.tile.rows_lo = 1;
  }
  if (most >= (usz)p.tile.rows_lo) {
    p.tile.rows_hi = 0x7fffffff;
    p.tile.tokens = AP_TILE_ROWS / 2 / (int)group * 2;
    p.tile.block_log2 = AP_TILE_BLOCK_LOG2;
    p.tile.ctas = std::min(base.sm_count, AP_MAX_CTAS);
    line_scale(&p.tile, nt, nseq, slots, 512, 512);
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
  if (!op) return fail(OPS_ARGS_NOT_SUPPORT, "null handle");
  const OpBase &base = op->h.base;
  const PagedAttnPlan plan = attention_paged_plan(base, m.nh, m.paged.nkvh, m.dh, a->mask == OPS_MASK_CAUSAL, g.batch.max_seq, m.nt, m.paged.nseq,
                                                m.paged.width * m.paged.page);
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
  if (plan.tile.ctas) OPS_TRY(attention_paged_tile(tile, bf16, plan.few.ctas != 0, s));
  if (plan.few.ctas + plan.tile.ctas)
    return ap_launch_beside("attention_paged(join)", bf16 ? attention_paged_join_kernel<true> : attention_paged_join_kernel<false>,
                            JOIN_BLOCKS_PER_SM * base.sm_count, JOIN_THREADS, 0, s, true, few, tile, plan.few_rows, plan.part_dh);
  return OPS_OK;
}
