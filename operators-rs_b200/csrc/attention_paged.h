// attention_paged.h — what the kernels of attention_paged share: arguments, the way a CTA finds its share, parked parts.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"

namespace ops {

constexpr int AP_MAX_DH = 128;
constexpr int AP_MAX_GROUP = 128;
constexpr int AP_MAX_CTAS = 256;  // of a kernel: the joining kernel holds a record of each
constexpr int AP_PAD = 4;  // a parked row: DH floats of unnormalised o, its reference point m and its sum l; 16-byte aligned

// What a CTA leaves for the kernel that joins the parts of units that several CTAs share.
struct __align__(16) PagedJoin {
  int ctas;                 // that have points of the unit this CTA has the first blocks of, and not the last: it and those behind it; else 0
  int row, tokens, head;    // of that unit: first row of the step, query tokens, kv head
  int front;                // whether this CTA's slot 0 holds a part (of the unit that its share begins in)
  int unused[3];
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

// Tensor maps over the whole cache, boxes of 64 columns x `rows` slots of one head of one page, 128-byte swizzle.
int attention_paged_maps(const PagedAttnArgs &a, bool bf16, uint32_t rows, CUtensorMap *k, CUtensorMap *v);
// A 4-d map of 16-bit elements, 64 of the innermost dim and `box1` x `box2` of the next two a box, 128-byte swizzle.
bool ap_encode(CUtensorMap *map, bool bf16, const void *ptr, const usz (&dims)[4], const isz (&strides)[3], uint32_t box1, uint32_t box2);
int attention_paged_few(const PagedAttnArgs &a, int rows, bool bf16, cudaStream_t s);
int attention_paged_few_ctas(const OpBase &base);
// beside: it may start while the launch in front of it, the few-rows kernel's, still runs; it ends behind it all the same.
int attention_paged_tile(const PagedAttnArgs &a, bool bf16, bool beside, cudaStream_t s);
constexpr int AP_FEW_BLOCK_LOG2 = 5, AP_FEW_BLOCK = 32, AP_TILE_BLOCK_LOG2 = 7, AP_TILE_BLOCK = 128;  // keys of a block
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

// CTA `cta`'s share of the line, by one warp: the points of all sequences, then the one its share begins in.  `report` says
// whether this CTA is the one that looks for what is wrong with the batch.  All lanes get the answer (at == end: nothing).
__device__ __forceinline__ void paged_locate(const PagedBatch &b, const PagedLine &l, int cta, bool report, PagedWalk *walk, int *total_out) {
  const int lane = threadIdx.x & 31;
  walk->seq = walk->begin = walk->at = walk->end = 0;
  *total_out = 0;
  long long sum = 0;
  int lo = 0, hi = 0, before = 0;
  // two passes through one copy of the code: all sequences for the sum, then up to the one that is looked for
  bool looking = false;
#pragma unroll 1
  for (int i0 = 0; i0 < b.nseq;) {
    const int i = i0 + lane;
    long long cost = 0;
    if (i < b.nseq) cost = (long long)paged_span(l, paged_seq(b, i, report && !looking)).head * l.nkvh;
    i0 += 32;
    if (!looking) {
      sum += cost;
      if (i0 < b.nseq) continue;
      // (a lane's sum stays below 2^47: 2^16 sequences of 2^31 points; its halves add up in 32 bits)
      sum = (long long)__reduce_add_sync(0xffffffffu, (unsigned)(sum & 0xffffff)) + ((long long)__reduce_add_sync(0xffffffffu, (unsigned)(sum >> 24)) << 24);
      // sequences that share rows (seq_start falls) can put more on the line than the host allowed for: nothing is done then
      const int total = sum <= 0x7fffffff ? (int)sum : 0;
      if (report && total != sum && lane == 0) atomicCAS(b.status, 0, OPS_PAGED_BAD_ROWS);
      *total_out = total;
      lo = paged_cut(l, total, cta);
      hi = paged_cut(l, total, cta + 1);
      if (lo >= hi) return;
      looking = true;
      i0 = 0;
      if (b.nseq > 32) continue;
      i0 = 32;  // of up to 32 sequences the costs are at hand
    }
    int upto = (int)cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned here = __ballot_sync(0xffffffffu, before + upto - (int)cost <= lo && lo < before + upto);
    if (here) {
      const int at = __ffs(here) - 1;
      walk->seq = i0 - 32 + at;
      walk->begin = before + __shfl_sync(0xffffffffu, upto - (int)cost, at);
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  walk->at = lo;
  walk->end = hi;
}

// By one thread.
__device__ __forceinline__ PagedPiece paged_step(const PagedBatch &b, const PagedLine &l, PagedWalk &w) {
  return paged_next(l, b.nseq, w, [&](int i) { return paged_seq(b, i, false); });
}

// The CTA's record for the joining kernel, written by one thread: `last` is the last piece of its share (its unit goes on in the
// next CTAs' shares if it is not the end of it), or seq < 0; front: its first piece is not the beginning of a unit.
__device__ __forceinline__ void paged_note_join(const PagedAttnArgs &a, int cta, const PagedPiece &last, bool front, int total) {
  PagedJoin j;
  memset(&j, 0, sizeof(j));
  j.front = front;
  if (last.seq >= 0 && last.lo == 0 && last.hi < last.blocks) {
    j.ctas = paged_first_behind(a.line, total, last.begin + last.cost) - cta;
    j.row = last.s.row + last.tile * a.line.tokens;
    j.tokens = min(a.line.tokens, last.s.n - last.tile * a.line.tokens);
    j.head = last.head;
  }
  a.joins[cta] = j;
}

// A launch may start while the one in front of it still runs (programmatic dependent launch): the front one says when the other
// may come, the other waits for all of its results.
__device__ __forceinline__ void pdl_let_next_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait_for_front() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

#ifdef __CUDACC__
// A launch, with `beside` one that may start while the one in front of it in the stream still runs.
template <class Kernel, class... Args>
int ap_launch_beside(const char *what, Kernel kernel, int grid, int block, int bytes, cudaStream_t s, bool beside, const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = (size_t)bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = beside ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(OPS_EXECUTION_FAILED, "%s: %s", what, cudaGetErrorString(e));
  return OPS_OK;
}
#endif

}  // namespace ops
