// attention_paged.h — what the kernels of attention_paged share: arguments, the way a CTA finds its share, parked parts.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"

namespace ops {

constexpr int AP_MAX_DH = 128;
constexpr int AP_MAX_GROUP = 128;
constexpr int AP_MAX_CTAS = 256;  // of a kernel
constexpr int AP_SHARES = 16;     // the few-rows kernel gets k / 16 of the CTAs where both kernels have work
constexpr int AP_FEW_JOIN = 16, AP_LEVELS = 2;  // parts are joined in groups, the groups in turn: 16^2 is AP_MAX_CTAS

struct PagedAttnArgs {
  const char *q, *k, *v;
  char *o;
  long long q_h, q_t, o_h, o_t;                  // byte strides: head, token
  long long kp_p, kp_h, kp_s, vp_p, vp_h, vp_s;  // byte strides: page, head, slot
  int nh, dh;
  float scale_log2;  // scale * log2(e): the softmax runs in powers of two
  PagedBatch batch;
  PagedLine line;
  uint32_t *arrived;  // [AP_LEVELS][line.ctas][8]: parts of a group that are parked; zero when the launch begins
  // parked parts, [2 * line.ctas, and line.ctas more for the few-rows kernel][rows of a unit]: unnormalised o, DH floats in whole
  // lines, and (m, l), its reference point and sum
  float *parts;
  float2 *parts_ml;
  PagedLine beside;             // the other kernel's line; ctas == 0: not launched
  PagedDiv by_ctas[AP_SHARES];  // by the CTAs that this kernel takes of a launch of both, by paged_share
};

// The few-rows kernel's CTAs for k of 16 shares; the tile kernel gets the others.
OPS_HD int paged_share(int ctas, int k) { return ctas * k / AP_SHARES > 0 ? ctas * k / AP_SHARES : 1; }

// Tensor maps over the whole cache, boxes of 64 columns x `rows` slots of one head of one page, 128-byte swizzle.
int attention_paged_maps(const PagedAttnArgs &a, bool bf16, uint32_t rows, CUtensorMap *k, CUtensorMap *v);
// A 4-d map of 16-bit elements, 64 of the innermost dim and `box1` x `box2` of the next two a box, 128-byte swizzle.
bool ap_encode(CUtensorMap *map, bool bf16, const void *ptr, const usz (&dims)[4], const isz (&strides)[3], uint32_t box1, uint32_t box2);
int attention_paged_few(const PagedAttnArgs &a, int rows, bool bf16, std::atomic<unsigned> &prepared, cudaStream_t s);
int attention_paged_few_ctas(const OpBase &base);
int attention_paged_tile(const PagedAttnArgs &a, bool bf16, bool behind_clear, std::atomic<unsigned> &prepared, cudaStream_t s);
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

// CTA `cta`'s share of the line, for its warp `finder`: the points of all sequences, then the one its share begins in (at == end:
// nothing).  Up to 32 sequences are that warp's alone; of more, every warp of the CTA adds up an even part first and the finder
// looks for its sequence in one of the parts: all warps of the CTA call, and meet once.  (One warp alone took a round trip to
// memory per 32 sequences, twice: 30 us of 2048 decoding requests' 116.)  `report` says whether this CTA is the one that looks
// for what is wrong with the batch.
//
// Where the line of the other kernel is not empty either, the two split the CTAs, and the SMs with them: the tile kernel's start on the
// SMs that the few-rows kernel leaves.  One after the other, the first would leave the tensor cores idle and the second the memory;
// and of the 148 SMs 96 are enough to read as fast as all (72: 89 %, 48: 63 %).  The split makes both take as long, by what a key costs
// an SM: 4 dh bytes at 68 GB/s, or 4 dh flops for each of 256 rows at 7 TFLOP/s, 2.5 times as long (a chunk of 487 tokens beside 31
// single ones over up to 2900 keys: 72 us, 86 one after the other).  Short sequences are bound by their number, not by the
// memory, and gain nothing from fewer SMs (512 single tokens over 100 keys beside eight prompts of 700 tokens: 72 us, 66 one after
// the other): then only a small share of the work runs beside the other's (64 of them: 47 us, 53 one after the other).  `l` comes
// back with its CTAs.
template <int WARPS, bool FEW>
__device__ __forceinline__ void paged_locate(const PagedAttnArgs &a, PagedLine &l, int cta, bool report, int warp, int finder, PagedWalk *walk, int *total_out) {
  static_assert(WARPS <= 32, "a lane per part");
  __shared__ int parts[3][WARPS];  // points of the line (-1: too many), of the other in 64s, sequences with a few rows
  const PagedBatch &b = a.batch;
  const bool both = a.beside.ctas > 0;
  const int lane = threadIdx.x & 31;
  walk->seq = walk->begin = walk->at = walk->end = 0;
  *total_out = 0;
  const bool together = b.nseq > 32;
  if (!together && warp != finder) return;
  const int part = together ? (b.nseq + WARPS * 32 - 1) / (WARPS * 32) * 32 : 32;
  int i0 = together ? warp * part : 0, end = min(b.nseq, i0 + part);
  long long sum = 0, sum_beside = 0;
  int few_seqs = 0;
  int lo = 0, before = 0;
  auto all_lanes = [](long long x) -> long long {  // the sum of non-negative numbers
    x = min(x, 1ll << 40);  // far more than a line holds; the halves of 32 such sums add up in 32 bits
    return (long long)__reduce_add_sync(0xffffffffu, (unsigned)(x & 0xffffff)) + ((long long)__reduce_add_sync(0xffffffffu, (unsigned)(x >> 24)) << 24);
  };
  bool looking = false, picking = false;  // for a sequence, for a part; both passes run through one copy of the code
#pragma unroll 1
  while (true) {
    const int i = i0 + lane;
    long long cost = 0;
    if (i < end) {
      const PagedSeq s = paged_seq(b, i, report && !looking);
      cost = (long long)paged_span(l, s).head * l.nkvh;
      if (both && !looking) {
        const long long other = (long long)paged_span(a.beside, s).head * l.nkvh;
        sum_beside += other;
        few_seqs += (FEW ? cost : other) > 0;
      }
    }
    i0 += 32;
    if (!looking) {
      sum += cost;
      if (i0 < end) continue;
      sum = all_lanes(sum);
      int mine = (int)sum, theirs = 0;
      if (both) {  // to weigh the two lines against each other: near enough
        theirs = __reduce_add_sync(0xffffffffu, (int)(sum_beside >> 6));
        few_seqs = __reduce_add_sync(0xffffffffu, few_seqs);
      }
      if (together) {
        if (lane == 0) {
          parts[0][warp] = sum <= 0x7fffffff ? mine : -1;
          parts[1][warp] = theirs;
          parts[2][warp] = few_seqs;
        }
        __syncthreads();
        if (warp != finder) return;
        mine = lane < WARPS ? parts[0][lane] : 0;
        sum = all_lanes(mine < 0 ? 1ll << 40 : mine);
        if (both) {
          theirs = __reduce_add_sync(0xffffffffu, lane < WARPS ? parts[1][lane] : 0);
          few_seqs = __reduce_add_sync(0xffffffffu, lane < WARPS ? parts[2][lane] : 0);
        }
      }
      // sequences that share rows (seq_start falls) can put more on the line than the host allowed for: nothing is done then
      const int total = sum <= 0x7fffffff ? (int)sum : 0;
      if (report && total != sum && lane == 0) atomicCAS(b.status, 0, OPS_PAGED_BAD_ROWS);
      *total_out = total;
      if (both && total > 0 && theirs > 0) {
        const float here = (float)total * (float)(1u << l.shift), there = (float)theirs * 64.f * (float)(1u << a.beside.shift);
        const float few = FEW ? here : there, tile = 2.5f * (FEW ? there : here);  // in what a key costs the few-rows kernel
        if (few >= 768.f * (float)few_seqs * (float)l.nkvh || 13.f * few <= 3.f * tile) {  // 640 keys a unit and more, or 3 / 16 of the work
          const int k = min(max(__float2int_rn(AP_SHARES * few / (few + tile)), 1), AP_SHARES * 3 / 4);
          l.ctas = FEW ? paged_share(l.ctas, k) : l.ctas - paged_share(l.ctas, k);
          l.by_ctas = a.by_ctas[k];
        }
      }
      if (cta >= l.ctas) return;
      lo = paged_cut(l, total, cta);
      const int hi = paged_cut(l, total, cta + 1);
      if (lo >= hi) return;
      walk->at = lo;
      walk->end = hi;
      looking = true;
      picking = together;
      if (picking) cost = mine;
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
      before += __shfl_sync(0xffffffffu, upto - (int)cost, at);
      if (!picking) {
        walk->seq = i0 - 32 + at;
        walk->begin = before;
        break;
      }
      picking = false;
      i0 = at * part;
      end = min(b.nseq, i0 + part);
      continue;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// By one thread.
__device__ __forceinline__ PagedPiece paged_step(const PagedBatch &b, const PagedLine &l, PagedWalk &w) {
  return paged_next(l, b.nseq, w, [&](int i) { return paged_seq(b, i, false); });
}

// Whether all parts but the caller's of a group are parked: then the caller's need not be.  One warp; what the others have
// written can be read behind it.
__device__ __forceinline__ bool paged_others_parked(const uint32_t *arrived, int group) {
  uint32_t n = 0;
  if ((threadIdx.x & 31) == 0) asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(arrived) : "memory");
  const bool all = __shfl_sync(0xffffffffu, n, 0) == (uint32_t)(group - 1);
  if (all) __threadfence();
  return all;
}
// The caller's warp has parked its part: the count as it was before.
__device__ __forceinline__ uint32_t paged_arrive(uint32_t *arrived) {
  __threadfence();
  __syncwarp();
  uint32_t before = 0;
  if ((threadIdx.x & 31) == 0) before = atomicAdd(arrived, 1u);
  return __shfl_sync(0xffffffffu, before, 0);
}
// ... whether it was the last of the group, as above.
__device__ __forceinline__ bool paged_arrive_last(uint32_t *arrived, int group) {
  const bool last = paged_arrive(arrived) == (uint32_t)(group - 1);
  if (last) __threadfence();
  return last;
}

// A launch may start while the one in front of it still runs (programmatic dependent launch): the front one says when the other
// may come, the other waits for all of its results.
__device__ __forceinline__ void pdl_let_next_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait_for_front() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

#ifdef __CUDACC__
// A launch with `bytes` of shared memory that may start while the one in front of it in the stream still runs.  `prepared`, the
// handle's: bits of the kernels that have been told how much (`bit`: this one's).
template <class Kernel, class... Args>
int ap_launch_beside(const char *what, std::atomic<unsigned> &prepared, unsigned bit, Kernel kernel, int grid, int block, int bytes, cudaStream_t s, const Args &...args) {
  cudaError_t e = cudaSuccess;
  if (!(prepared.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) prepared.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = (size_t)bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) return OPS_OK;
  cudaGetLastError();  // not the next launch's to answer for
  return fail(OPS_EXECUTION_FAILED, "%s: %s", what, cudaGetErrorString(e));
}
#endif

}  // namespace ops
