// rope_norm.cu — heads of the new tokens normalised and rotated in one pass, in place of a norm launch and a rope launch
// (ops_rope_norm_launch), and the same with the keys and values going straight into a paged cache (ops_kv_append_paged_launch).
// Neither has a counterpart in the crate; the rotation is rope's (operators/src/rope/common_cpu/mod.rs:164-202: adjacent pairs),
// the norm rms_norm's (operators/src/rms_norm/common_cpu/mod.rs:28-93) over one head.
//
//   r = 1 / sqrt(mean_d x[d]^2 + eps);  n[d] = x[d] r w[h, d];  a_k = pos theta^(-2k/dh)
//   y[2k] = n[2k] cos a_k - n[2k+1] sin a_k;  y[2k+1] = n[2k] sin a_k + n[2k+1] cos a_k
//
// HBM-bound: every head vector is read once and written once, 4 dh bytes a head.  A lane holds 8 consecutive elements (one
// 128-bit access), so a head takes dh / 8 lanes (rounded up to a power of two) and its sum of squares a few shuffles.  A warp
// walks heads of ONE token: the lane's four (sin, cos) are the same for all of them and are computed once, in registers, with no
// shared memory and no barrier; two or four vectors are in flight per lane.  With few tokens the heads of a token are dealt to
// several warps, so that a decode step fills the machine.  Everything is f32 and rounded once; the angle is taken in turns,
// pos * (theta^(-2k/dh) / 2 pi), in f64 and reduced there: in f32 it would be off by pos * 2^-24 rad.
// What bounded it first was instruction issue (full-range sincospi, 64-bit address arithmetic per vector: 70 us for 8192 rows of
// 40 heads of 128); with angles reduced in f64 in front of the special-function unit, pointers that step and packed f32 pairs
// it streams: 33 us.  The norm was 5 us of that, each vector's chain of shuffles behind the last one's: with the sums of a round
// side by side 30 us, 5.6 TB/s (6 blocks an SM; with 7, or the weights loaded ahead of the sums, registers spill: 31, 37 us).  The
// append takes 7 blocks all the same: in rounds of four with norms it spills (32 to 46 bytes of stores, 76 to 88 of loads a thread, at
// 72 registers), and seven prompts take 30.4 us against 31.2 with 6.  Reads and writes both bypass what other kernels keep in
// L2 (either alone changed nothing for these kernels; the attention behind an append was not timed with them).
#include <type_traits>

#include "device_utils.cuh"
#include "internal.h"
#include "paged.h"

namespace ops {

constexpr int RN_MAX_PAIRS = 128;  // dh <= 256
constexpr int RN_WARPS = 4;

struct RotateTurns {
  double v[RN_MAX_PAIRS];  // theta^(-2k/dh) / 2 pi
};

struct RotateArgs {
  // byte strides: token, head
  const char *q, *k, *v;
  char *qo;
  long long q_t, q_h, k_t, k_h, v_t, v_h, qo_t, qo_h;
  const void *pos;
  long long pos_t;
  int pos64;
  const char *w;  // null: no norm
  long long w_h;
  float eps, inv_dh;
  int nt, nh, nkvh;     // without APPEND nkvh = 0
  int dh, lanes;        // lanes of a warp that hold one head: dh / 8 rounded up to a power of two
  int slices, per_slice;  // warps per token, heads each of them walks
  // APPEND
  char *k_pages, *v_pages;
  long long kp_p, kp_h, kp_s, vp_p, vp_h, vp_s;  // byte strides: page, head, slot
  PagedBatch batch;
};

// 8 consecutive elements as pairs of f32
__device__ __forceinline__ void pairs_of(uint4 v, float2 (&f)[4], __half) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __half22float2(h[e]);
}
__device__ __forceinline__ void pairs_of(uint4 v, float2 (&f)[4], __nv_bfloat16) {
  const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __bfloat1622float2(h[e]);
}
// ... of a row of weights, as they are loaded
template <class T> struct RowPiece {
  typedef uint4 type;
};
struct __align__(16) EightFloats {
  float v[8];
};
template <> struct RowPiece<float> {
  typedef EightFloats type;
};
__device__ __forceinline__ void pairs_of(const EightFloats &v, float2 (&f)[4], float) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = make_float2(v.v[2 * e], v.v[2 * e + 1]);
}
__device__ __forceinline__ uint32_t pair_to(float2 v, __half) {
  const __half2 h = __float22half2_rn(v);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pair_to(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(v);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <class E, class W, bool NORM, bool APPEND, int RN_UNROLL>
__global__ void __launch_bounds__(RN_WARPS * 32, APPEND ? 7 : 6) rotate_heads_kernel(const __grid_constant__ RotateArgs a, const __grid_constant__ RotateTurns turns) {
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * RN_WARPS + (threadIdx.x >> 5);
  if (APPEND) {
    // What is wrong with the batch, a lane per sequence: rows alone do not show it (none may find its way to a sequence whose
    // start falls).  Warps that have no sequence, nearly all, go on at once.
    for (long long i = item * 32 + lane; i < a.batch.nseq; i += (long long)gridDim.x * (RN_WARPS * 32)) paged_seq(a.batch, (int)i, true);
  }
  const int tok = (int)(item / a.slices), slice = (int)(item - (long long)tok * a.slices);
  if (tok >= a.nt) return;
  const int sub = lane & (a.lanes - 1);   // which 8 elements of the head
  const int first = lane / a.lanes;       // which of the heads that the warp holds at a time
  const int at_once = 32 / a.lanes;
  const bool active = sub * 8 < a.dh;
  const int heads = a.nh + (APPEND ? 2 * a.nkvh : 0);
  const int h_begin = slice * a.per_slice, h_end = min(heads, h_begin + a.per_slice);

  if (APPEND) {  // rows of nobody are left as they are
    const uint32_t lo = a.batch.start[0], hi = a.batch.start[a.batch.nseq];
    if ((uint32_t)tok < lo || (uint32_t)tok >= hi) return;
  }
  const double pos = a.pos64 ? (double)*reinterpret_cast<const unsigned long long *>(reinterpret_cast<const char *>(a.pos) + tok * a.pos_t)
                             : (double)*reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(a.pos) + tok * a.pos_t);
  float sn[4], cs[4];
  bool turned = false;
  auto turn = [&]() {
    if (turned) return;
    turned = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // reduced to half a turn either way in f64; the special-function unit is off by less than 2^-20 there, a five-hundredth
      // of the 16-bit result's half step
      const double t = pos * turns.v[min(sub * 4 + e, RN_MAX_PAIRS - 1)];
      __sincosf(6.283185307f * (float)(t - rint(t)), &sn[e], &cs[e]);
    }
  };

  // Heads [lo, hi) of one operand, counted from its first head; dst null: nowhere to write.  The loads of a round are issued before
  // the first is used, those of the first round before the angles are there.
  auto walk = [&](const char *src, long long src_h, char *dst, long long dst_h, const char *w, int lo, int hi, auto rotated) {
    if (lo >= hi) return;
    src += (long long)(lo + first) * src_h + sub * 16;
    dst += (long long)(lo + first) * dst_h + sub * 16;
    if (NORM) w += (long long)(lo + first) * a.w_h + sub * 8 * (int)sizeof(W);
    const long long src_step = at_once * src_h, dst_step = at_once * dst_h, w_step = at_once * a.w_h;
    for (int h = lo + first; h - first < hi; h += at_once * RN_UNROLL) {
      uint4 x[RN_UNROLL];
#pragma unroll
      for (int u = 0; u < RN_UNROLL; ++u) {
        x[u] = make_uint4(0, 0, 0, 0);
        if (active && h + u * at_once < hi) x[u] = ld_stream_16(src + u * src_step);
      }
      if (rotated) turn();
      // the sums of a round side by side: the shuffles of a step wait together, not in turn
      float r[RN_UNROLL];
      if (rotated && NORM) {
#pragma unroll
        for (int u = 0; u < RN_UNROLL; ++u) {
          float2 f[4];
          pairs_of(x[u], f, E());
          float2 ss = __fmul2_rn(f[0], f[0]);
#pragma unroll
          for (int e = 1; e < 4; ++e) ss = __ffma2_rn(f[e], f[e], ss);
          r[u] = ss.x + ss.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          if (o < a.lanes) {
#pragma unroll
            for (int u = 0; u < RN_UNROLL; ++u) r[u] += __shfl_xor_sync(0xffffffffu, r[u], o);
          }
#pragma unroll
        for (int u = 0; u < RN_UNROLL; ++u) r[u] = rsqrtf(fmaf(r[u], a.inv_dh, a.eps));
      }
#pragma unroll
      for (int u = 0; u < RN_UNROLL; ++u) {
        const bool there = active && h + u * at_once < hi;
        if (rotated) {
          float2 f[4];
          pairs_of(x[u], f, E());
          if (NORM) {
            float2 wt[4];
            typename RowPiece<W>::type weight = typename RowPiece<W>::type();
            if (there) weight = *reinterpret_cast<const typename RowPiece<W>::type *>(w + u * w_step);
            pairs_of(weight, wt, W());
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = __fmul2_rn(f[e], __fmul2_rn(wt[e], make_float2(r[u], r[u])));
          }
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y[e] = pair_to(make_float2(f[e].x * cs[e] - f[e].y * sn[e], f[e].x * sn[e] + f[e].y * cs[e]), E());
          x[u] = make_uint4(y[0], y[1], y[2], y[3]);
        }
        if (there) st_stream_16(dst + u * dst_step, x[u]);
      }
      src += RN_UNROLL * src_step;
      dst += RN_UNROLL * dst_step;
      if (NORM) w += RN_UNROLL * w_step;
    }
  };
  walk(a.q + (long long)tok * a.q_t, a.q_h, a.qo + (long long)tok * a.qo_t, a.qo_h, a.w, h_begin, min(h_end, a.nh), std::true_type());
  if (!APPEND || h_end <= a.nh) return;

  // the token's slot in the cache
  const int i = paged_find(a.batch, (uint32_t)tok);
  if (i < 0) return;
  const PagedSeq s = paged_seq(a.batch, i, false);
  const long long slot = (long long)a.batch.len[i] - s.n + (tok - s.row);  // by the length as given: a cut one would move the token
  int wrong = 0;
  uint32_t page = 0;
  if (tok - s.row >= s.n) {
    wrong = OPS_PAGED_BAD_ROWS;
  } else if (slot < 0 || slot >= ((long long)a.batch.width << a.batch.page_log2)) {
    wrong = OPS_PAGED_BAD_LENGTH;
  } else {
    page = a.batch.table[(long long)i * a.batch.table_ld + (slot >> a.batch.page_log2)];
    if (page >= a.batch.npages) wrong = OPS_PAGED_BAD_PAGE;
  }
  if (wrong) {
    if (lane == 0) atomicCAS(a.batch.status, 0, wrong);
    return;
  }
  const int at = (int)slot & ((1 << a.batch.page_log2) - 1);
  walk(a.k + (long long)tok * a.k_t, a.k_h, a.k_pages + (long long)page * a.kp_p + (long long)at * a.kp_s, a.kp_h,
       NORM ? a.w + (long long)a.nh * a.w_h : nullptr, max(0, h_begin - a.nh), min(h_end - a.nh, a.nkvh), std::true_type());
  walk(a.v + (long long)tok * a.v_t, a.v_h, a.v_pages + (long long)page * a.vp_p + (long long)at * a.vp_s, a.vp_h, nullptr,
       max(0, h_begin - a.nh - a.nkvh), min(h_end - a.nh - a.nkvh, a.nkvh), std::false_type());
}

// (Sixty-four calls of pow are a third of what a small launch costs the host: a thread keeps the last table it made.)
static const RotateTurns &rotate_turns(float theta, usz dh) {
  static thread_local RotateTurns t;
  static thread_local float for_theta = 0.f;
  static thread_local usz for_dh = 0;
  if (for_dh != dh || memcmp(&for_theta, &theta, sizeof(theta)) != 0) {
    for (int k = 0; k < RN_MAX_PAIRS; ++k)
      t.v[k] = (usz)k < dh / 2 ? std::pow((double)theta, -2.0 * k / (double)dh) / 6.283185307179586476925 : 0.0;
    for_theta = theta;
    for_dh = dh;
  }
  return t;
}

// Warps per token.  About 16 warps an SM hide a round trip to memory; with no more than that, and few heads a warp, a round of two
// vectors a lane is enough (a round of four spends instructions on vectors that are not there: 64 rows of 40 heads 3.8 against
// 3.2 us, 1777 rows of 5 heads 5.5 against 4.4).  Otherwise a warp walks a whole token in rounds of four, or half of one as long
// as that makes no more than 48 warps an SM (8192 rows of 40 heads: 29.9 us against 33.3 with twice the warps; ragged prompts of
// 48 heads: 30.2 us against 32.6 with 32 warps an SM; rounds of two were a tenth slower in both).
static int rotate_split(const OpBase &base, RotateArgs *a, int heads) {
  a->lanes = 1;
  while (a->lanes * 8 < a->dh) a->lanes *= 2;
  const int at_once = 32 / a->lanes, passes = (heads + at_once - 1) / at_once;
  auto split = [&](long long per_sm) {
    const long long most = std::min<long long>(passes, std::max<long long>(1, (per_sm * base.sm_count + a->nt - 1) / a->nt));
    const int each = (int)((passes + most - 1) / most);
    a->per_slice = each * at_once;
    a->slices = (passes + each - 1) / each;
    return each;
  };
  if (split(16) <= 4) return 2;
  split(48);
  return 4;
}

template <bool APPEND, int RN_UNROLL>
static int rotate_launch(const char *what, const RotateArgs &a, const RotateTurns &turns, bool bf16, uint32_t w_dt, cudaStream_t s) {
  const unsigned long long items = (unsigned long long)a.nt * a.slices;
  const unsigned grid = (unsigned)((items + RN_WARPS - 1) / RN_WARPS);
#define RN_GO(E, W, NORM) rotate_heads_kernel<E, W, NORM, APPEND, RN_UNROLL><<<grid, RN_WARPS * 32, 0, s>>>(a, turns)
  if (!a.w) {
    if (bf16) RN_GO(__nv_bfloat16, float, false);
    else RN_GO(__half, float, false);
  } else if (w_dt == OPS_DT_F32) {
    if (bf16) RN_GO(__nv_bfloat16, float, true);
    else RN_GO(__half, float, true);
  } else {
    if (bf16) RN_GO(__nv_bfloat16, __nv_bfloat16, true);
    else RN_GO(__half, __half, true);
  }
#undef RN_GO
  return check_launch(what);
}

// w [heads, dh] of type dt or f32, rows of 16-byte pieces; stride 0 shares a row
static int weight_checks(const char *op, const ops_layout *l, const void *base, uint32_t dt, usz heads, usz dh) {
  if (dyn(l->shape[0]) || dyn(l->shape[1]) || dyn(l->strides[0]) || dyn(l->strides[1]))
    return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: every shape and stride of w must be static at launch", op);
  if (l->dt != dt && l->dt != OPS_DT_F32) return fail(OPS_TYPE_NOT_SUPPORT, "%s: w must have the type of the heads or f32", op);
  if (l->shape[0] != heads || l->shape[1] != dh) return fail(OPS_SHAPE_MISMATCH, "%s: w must be [%zu, %zu]", op, heads, dh);
  if (l->strides[1] != (isz)dt_size(l->dt) || (heads > 1 && l->strides[0] % 16) || !aligned(base, 16))
    return fail(OPS_STRIDES_NOT_SUPPORT, "%s: rows of w must be contiguous and 16-byte aligned", op);
  return OPS_OK;
}

// p [nt], u32 or u64
static int pos_checks(const char *op, const ops_layout *l, const void *base) {
  if (dyn(l->shape[0]) || dyn(l->strides[0])) return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: shape and stride of p must be static at launch", op);
  if (l->shape[0] > 1 && l->strides[0] % (isz)dt_size(l->dt)) return fail(OPS_STRIDES_NOT_SUPPORT, "%s: stride of p must be a multiple of its element", op);
  if (!base) return fail(OPS_DYNAMIC_NOT_SUPPORT, "%s: null base pointer of p at launch", op);
  if (!aligned(base, dt_size(l->dt))) return fail(OPS_STRIDES_NOT_SUPPORT, "%s: p must be aligned to its element", op);
  return OPS_OK;
}

static int rope_norm_meta(const ops_rope_norm_args *a, usz *nt, usz *nh, usz *dh) {
  if (a->y_layout.ndim != 3) return fail(OPS_RANK_NOT_SUPPORT, "y.ndim = %u, 3 expected", a->y_layout.ndim);
  if (a->x_layout.ndim != 3) return fail(OPS_RANK_NOT_SUPPORT, "x.ndim = %u, 3 expected", a->x_layout.ndim);
  if (a->p_layout.ndim != 1) return fail(OPS_RANK_NOT_SUPPORT, "p.ndim = %u, 1 expected", a->p_layout.ndim);
  if (a->w_layout.ndim != 2) return fail(OPS_RANK_NOT_SUPPORT, "w.ndim = %u, 2 expected", a->w_layout.ndim);
  if (a->y_layout.dt != a->x_layout.dt) return fail(OPS_TYPE_MISMATCH, "element types of y and x differ");
  if (a->p_layout.dt != OPS_DT_U32 && a->p_layout.dt != OPS_DT_U64) return fail(OPS_TYPE_NOT_SUPPORT, "data type of p is not supported, must be u32 or u64");
  const usz nts[3] = {a->y_layout.shape[0], a->x_layout.shape[0], a->p_layout.shape[0]};
  const usz nhs[3] = {a->y_layout.shape[1], a->x_layout.shape[1], a->w_layout.shape[0]};
  const usz dhs[3] = {a->y_layout.shape[2], a->x_layout.shape[2], a->w_layout.shape[1]};
  if (!merge_dims(nts, 3, nt)) return fail(OPS_SHAPE_MISMATCH, "nt of y, x and p differ");
  if (!merge_dims(nhs, 3, nh)) return fail(OPS_SHAPE_MISMATCH, "nh of y, x and w differ");
  if (!merge_dims(dhs, 3, dh)) return fail(OPS_SHAPE_MISMATCH, "dh of y, x and w differ");
  return OPS_OK;
}

int rope_norm_enqueue(const OpBase *base, const ops_rope_norm_args *a, cudaStream_t s) {
  usz nt = 0, nh = 0, dh = 0;
  OPS_TRY(rope_norm_meta(a, &nt, &nh, &dh));
  static const char *op = "rope_norm";
  const uint32_t dt = a->x_layout.dt;
  if (dyn(a->epsilon) || dyn(a->theta)) return fail(OPS_DYNAMIC_NOT_SUPPORT, "rope_norm: epsilon and theta must be static at launch");
  // everything this pass does not take is answered with ArgsNotSupport: rms_norm and rope chained do the same
  const ops_layout *ls[2] = {&a->y_layout, &a->x_layout};
  const void *bases[2] = {a->y_base, a->x_base};
  static const char *names[2] = {"y", "x"};
  bool chain = dt != OPS_DT_F16 && dt != OPS_DT_BF16;
  for (int i = 0; i < 2; ++i) {
    const int rc = rows16_checks(op, names[i], ls[i], bases[i], true);
    if (rc == OPS_STRIDES_NOT_SUPPORT) chain = true;
    else if (rc != OPS_OK) return rc;
  }
  if (nt == 0 || nh == 0 || dh == 0) return OPS_OK;
  if (!a->w_base) return fail(OPS_DYNAMIC_NOT_SUPPORT, "rope_norm: null base pointer of w at launch");
  const int rw = weight_checks(op, &a->w_layout, a->w_base, dt, nh, dh);
  if (rw == OPS_STRIDES_NOT_SUPPORT) chain = true;
  else if (rw != OPS_OK) return rw;
  OPS_TRY(pos_checks(op, &a->p_layout, a->p_base));
  if (chain || dh % 8 || dh > 2 * RN_MAX_PAIRS)
    return fail(OPS_ARGS_NOT_SUPPORT, "rope_norm: needs f16 or bf16 rows, contiguous and 16-byte aligned, with dh a multiple of 8 (<= 256); chain rms_norm and rope instead");
  if (nt > 0x3fffffffu || nh > 0xffffu) return fail(OPS_SHAPE_NOT_SUPPORT, "rope_norm: shape too large");
  if (!base) return fail(OPS_ARGS_NOT_SUPPORT, "null handle");
  RotateArgs g;
  memset(&g, 0, sizeof(g));
  g.q = (const char *)a->x_base;
  g.q_t = a->x_layout.strides[0];
  g.q_h = a->x_layout.strides[1];
  g.qo = (char *)a->y_base;
  g.qo_t = a->y_layout.strides[0];
  g.qo_h = a->y_layout.strides[1];
  g.pos = a->p_base;
  g.pos_t = a->p_layout.strides[0];
  g.pos64 = a->p_layout.dt == OPS_DT_U64;
  g.w = (const char *)a->w_base;
  g.w_h = a->w_layout.strides[0];
  g.eps = a->epsilon;
  g.nt = (int)nt;
  g.nh = (int)nh;
  g.dh = (int)dh;
  g.inv_dh = 1.f / (float)dh;
  const int unroll = rotate_split(*base, &g, (int)nh);
  if ((unsigned long long)nt * g.slices > 0x7fffffffull) return fail(OPS_SHAPE_NOT_SUPPORT, "rope_norm: shape too large");
  DeviceGuard guard(base->device);
  return (unroll == 2 ? rotate_launch<false, 2> : rotate_launch<false, 4>)(op, g, rotate_turns(a->theta, dh), dt == OPS_DT_BF16, a->w_layout.dt, s);
}

struct AppendMeta {
  uint32_t dt;
  usz nt, nh, nkvh, dh;
  PagedMeta paged;
};

static int append_meta(const ops_kv_append_paged_args *a, AppendMeta *m) {
  const ops_layout *ls[4] = {&a->q_out_layout, &a->q_layout, &a->k_layout, &a->v_layout};
  static const char *names[4] = {"q_out", "q", "k", "v"};
  for (int i = 0; i < 4; ++i)
    if (ls[i]->ndim != 3) return fail(OPS_RANK_NOT_SUPPORT, "%s.ndim = %u, 3 expected", names[i], ls[i]->ndim);
  if (a->p_layout.ndim != 1) return fail(OPS_RANK_NOT_SUPPORT, "p.ndim = %u, 1 expected", a->p_layout.ndim);
  if (a->w_base && a->w_layout.ndim != 2) return fail(OPS_RANK_NOT_SUPPORT, "w.ndim = %u, 2 expected", a->w_layout.ndim);
  OPS_TRY(paged_meta(&a->batch, &a->k_pages_layout, &a->v_pages_layout, &m->paged));
  m->dt = a->q_layout.dt;
  if (m->dt != OPS_DT_F16 && m->dt != OPS_DT_BF16) return fail(OPS_TYPE_NOT_SUPPORT, "kv_append_paged: f16 or bf16 expected");
  const uint32_t dts[5] = {a->q_out_layout.dt, a->k_layout.dt, a->v_layout.dt, a->k_pages_layout.dt, a->v_pages_layout.dt};
  for (int i = 0; i < 5; ++i)
    if (dts[i] != m->dt) return fail(OPS_TYPE_MISMATCH, "element types of q, q_out, k, v and the cache differ");
  if (a->p_layout.dt != OPS_DT_U32 && a->p_layout.dt != OPS_DT_U64) return fail(OPS_TYPE_NOT_SUPPORT, "data type of p is not supported, must be u32 or u64");
  const usz nts[5] = {ls[0]->shape[0], ls[1]->shape[0], ls[2]->shape[0], ls[3]->shape[0], a->p_layout.shape[0]};
  const usz nhs[2] = {ls[0]->shape[1], ls[1]->shape[1]};
  const usz nks[3] = {ls[2]->shape[1], ls[3]->shape[1], m->paged.nkvh};
  const usz dhs[5] = {ls[0]->shape[2], ls[1]->shape[2], ls[2]->shape[2], ls[3]->shape[2], m->paged.dh};
  if (!merge_dims(nts, 5, &m->nt)) return fail(OPS_SHAPE_MISMATCH, "nt of q, q_out, k, v and p differ");
  if (!merge_dims(nhs, 2, &m->nh)) return fail(OPS_SHAPE_MISMATCH, "nh of q and q_out differ");
  if (!merge_dims(nks, 3, &m->nkvh)) return fail(OPS_SHAPE_MISMATCH, "nkvh of k, v and the cache differ");
  if (!merge_dims(dhs, 5, &m->dh)) return fail(OPS_SHAPE_MISMATCH, "dh of q, q_out, k, v and the cache differ");
  if (!dyn(m->dh) && (m->dh % 8 || m->dh > 2 * RN_MAX_PAIRS)) return fail(OPS_SHAPE_NOT_SUPPORT, "kv_append_paged: dh = %zu, a multiple of 8 up to 256 expected", m->dh);
  if (!dyn(m->nt) && m->nt > 0x3fffffffu) return fail(OPS_SHAPE_NOT_SUPPORT, "kv_append_paged: too many rows");
  if (!dyn(m->nh) && m->nh > 0xffffu) return fail(OPS_SHAPE_NOT_SUPPORT, "kv_append_paged: too many heads");
  return OPS_OK;
}

}  // namespace ops

using namespace ops;

OPS_DEFINE_PAGED_HANDLE(kv_append_paged)

OPS_API int ops_kv_append_paged_scheme(ops_kv_append_paged *op, const ops_kv_append_paged_args *args, size_t max_ws, size_t *ws_out) {
  (void)op;
  (void)max_ws;
  AppendMeta m;
  OPS_TRY(append_meta(args, &m));
  if (ws_out) *ws_out = 0;
  return OPS_OK;
}

OPS_API int ops_kv_append_paged_launch(const ops_kv_append_paged *op, const ops_kv_append_paged_args *a, void *ws, size_t ws_len, void *stream) {
  (void)ws;
  (void)ws_len;
  static const char *name = "kv_append_paged";
  AppendMeta m;
  OPS_TRY(append_meta(a, &m));
  if (dyn(a->theta) || (a->w_base && dyn(a->epsilon))) return fail(OPS_DYNAMIC_NOT_SUPPORT, "kv_append_paged: epsilon and theta must be static at launch");
  RotateArgs g;
  memset(&g, 0, sizeof(g));
  const ops_layout *ls[4] = {&a->q_out_layout, &a->q_layout, &a->k_layout, &a->v_layout};
  const void *bases[4] = {a->q_out_base, a->q_base, a->k_base, a->v_base};
  static const char *names[4] = {"q_out", "q", "k", "v"};
  for (int i = 0; i < 4; ++i) OPS_TRY(rows16_checks(name, names[i], ls[i], bases[i], true));
  OPS_TRY(paged_launch_checks(name, &a->batch, &a->k_pages_layout, a->k_pages_base, &a->v_pages_layout, a->v_pages_base, m.paged, m.nt,
                              op ? op->h.status : nullptr, &g.batch));
  if (m.nt == 0 || m.dh == 0 || m.nh + m.nkvh == 0 || m.paged.nseq == 0) return OPS_OK;
  OPS_TRY(pos_checks(name, &a->p_layout, a->p_base));
  if (a->w_base) OPS_TRY(weight_checks(name, &a->w_layout, a->w_base, m.dt, m.nh + m.nkvh, m.dh));
  if (!op) return fail(OPS_ARGS_NOT_SUPPORT, "null handle");
  g.qo = (char *)a->q_out_base;
  g.qo_t = ls[0]->strides[0];
  g.qo_h = ls[0]->strides[1];
  g.q = (const char *)a->q_base;
  g.q_t = ls[1]->strides[0];
  g.q_h = ls[1]->strides[1];
  g.k = (const char *)a->k_base;
  g.k_t = ls[2]->strides[0];
  g.k_h = ls[2]->strides[1];
  g.v = (const char *)a->v_base;
  g.v_t = ls[3]->strides[0];
  g.v_h = ls[3]->strides[1];
  g.pos = a->p_base;
  g.pos_t = a->p_layout.strides[0];
  g.pos64 = a->p_layout.dt == OPS_DT_U64;
  g.w = (const char *)a->w_base;
  g.w_h = a->w_base ? a->w_layout.strides[0] : 0;
  g.eps = a->epsilon;
  g.nt = (int)m.nt;
  g.nh = (int)m.nh;
  g.nkvh = (int)m.nkvh;
  g.dh = (int)m.dh;
  g.k_pages = (char *)a->k_pages_base;
  g.v_pages = (char *)a->v_pages_base;
  const isz *sk = a->k_pages_layout.strides, *sv = a->v_pages_layout.strides;
  g.kp_p = sk[0];
  g.kp_h = sk[1];
  g.kp_s = sk[2];
  g.vp_p = sv[0];
  g.vp_h = sv[1];
  g.vp_s = sv[2];
  g.inv_dh = 1.f / (float)m.dh;
  const int unroll = rotate_split(op->h.base, &g, g.nh + 2 * g.nkvh);
  if ((unsigned long long)m.nt * g.slices > 0x7fffffffull) return fail(OPS_SHAPE_NOT_SUPPORT, "kv_append_paged: shape too large");
  DeviceGuard guard(op->h.base.device);
  return (unroll == 2 ? rotate_launch<true, 2> : rotate_launch<true, 4>)(name, g, rotate_turns(a->theta, m.dh), m.dt == OPS_DT_BF16, a->w_base ? a->w_layout.dt : (uint32_t)OPS_DT_F32, (cudaStream_t)stream);
}
