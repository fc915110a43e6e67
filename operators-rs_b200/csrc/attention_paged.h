// attention_paged.h — what the kernels of attention_paged share: arguments, the way a CTA finds its share, parked parts.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"

namespace ops {

constexpr int AP_MAX_DH = 128;
constexpr int AP_MAX_GROUP = 128;
constexpr int AP_MAX_CTAS = 1024;
constexpr int AP_PAD = 4;  // a parked row: DH floats of unnormalised o, its reference point m and its sum l; 16-byte aligned

// A unit that several CTAs share, as the one that has its first blocks writes it down for the kernel that joins the parts.
struct PagedJoin {
  int ctas;               // that have points of the unit, the writer and those behind it; 0: nothing to join
  int row, tokens, head;  // first row of the step, query tokens, kv head
  int blocks, active;     // of the unit; of the launch
  i64 begin, cost, total;  // unit on the line; points of the line
};

struct PagedAttnArgs {
  const char *q, *k, *v;
  char *o;
  long long q_h, q_t, o_h, o_t;                  // byte strides: head, token
  long long kp_p, kp_h, kp_s, vp_p, vp_h, vp_s;  // byte strides: page, head, slot
  int nh, dh;
  float scale_log2;  // scale * log2(e): the softmax runs in powers of two
  PagedBatch batch;
  PagedLine line;
  PagedJoin *joins;  // [line.ctas]
  float *parts;      // [2 * line.ctas][rows of a unit][DH + AP_PAD]
};

int attention_paged_few(const PagedAttnArgs &a, int rows, bool bf16, cudaStream_t s);
int attention_paged_few_ctas(const OpBase &base, int rows);
int attention_paged_tile(const PagedAttnArgs &a, bool bf16, cudaStream_t s);
constexpr int AP_FEW_BLOCK = 128, AP_TILE_BLOCK = 128;  // keys of a block of either kernel
constexpr int AP_TILE_ROWS = 256;                       // query rows of a unit of the tile kernel: two tiles

#ifdef __CUDACC__
__device__ __forceinline__ float ap_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF>
__device__ __forceinline__ uint32_t ap_pack(float lo, float hi) {  // first value in the low half
  if (BF) {
    __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&t);
  }
  __half2 t = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&t);
}

// CTA `cta`'s share of the line, found by all THREADS of a block together: a prefix sum over the sequences.  `report` says
// whether this block is the one that looks for what is wrong with the batch.  total: the line's points.
template <int THREADS>
__device__ PagedWalk paged_locate(const PagedBatch &b, const PagedLine &l, int cta, bool report, i64 *total_out) {
  __shared__ i64 warp_sums[THREADS / 32];
  __shared__ PagedWalk found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (b.nseq + THREADS - 1) / THREADS, i0 = min(b.nseq, (int)threadIdx.x * per), i1 = min(b.nseq, i0 + per);
  i64 mine = 0;
  for (int i = i0; i < i1; ++i) mine += paged_span(l, paged_seq(b, i, report)).head * l.nkvh;
  i64 upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const i64 x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  i64 total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w == warp) upto += total;
    total += warp_sums[w];
  }
  const int active = paged_active(l, total);
  *total_out = total;
  PagedWalk w;
  w.seq = 0;
  w.begin = w.at = w.end = 0;
  if (cta >= active) return w;  // the whole block
  const i64 lo = paged_cut(total, active, cta), hi = paged_cut(total, active, cta + 1);
  i64 begin = upto - mine;
  if (begin <= lo && lo < upto) {
    int i = i0;
    while (true) {
      const i64 all = paged_span(l, paged_seq(b, i, false)).head * l.nkvh;
      if (begin + all > lo) break;
      begin += all;
      ++i;
    }
    found.seq = i;
    found.begin = begin;
    found.at = lo;
    found.end = hi;
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ PagedPiece paged_step(const PagedBatch &b, const PagedLine &l, PagedWalk &w) {
  return paged_next(l, b.nseq, w, [&](int i) { return paged_seq(b, i, false); });
}

// The CTA's record for the joining kernel, written by one thread: `piece` is the last of its share (its unit goes on in the next
// CTAs' shares if it is not the end of it), or seq < 0.  walk: as the piece left it.
__device__ __forceinline__ void paged_note_join(const PagedAttnArgs &a, int cta, const PagedPiece &piece, const PagedWalk &walk, i64 total) {
  PagedJoin j;
  memset(&j, 0, sizeof(j));
  if (piece.seq >= 0 && piece.lo == 0 && piece.hi < piece.blocks) {
    const PagedSpan p = paged_span(a.line, piece.s);
    j.begin = walk.begin + piece.head * p.head + paged_tile_begin(a.line, p, piece.tile);
    j.cost = a.line.overhead + p.base + (i64)p.ramp * (piece.tile + 1);
    j.total = total;
    j.active = paged_active(a.line, total);
    j.ctas = paged_first_behind(total, j.active, j.begin + j.cost) - cta;
    j.row = piece.s.row + piece.tile * a.line.tokens;
    j.tokens = min(a.line.tokens, piece.s.n - piece.tile * a.line.tokens);
    j.head = piece.head;
    j.blocks = piece.blocks;
  }
  a.joins[cta] = j;
}

// A launch may start while the one in front of it still runs (programmatic dependent launch): the front one says when the other
// may come, the other waits for all of its results.
__device__ __forceinline__ void pdl_let_next_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait_for_front() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

}  // namespace ops
