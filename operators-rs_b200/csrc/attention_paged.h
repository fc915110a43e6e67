// attention_paged.h — what the kernels of attention_paged share: arguments, the way a CTA finds its share, parked parts.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"

namespace ops {

constexpr int AP_MAX_DH = 128;
constexpr int AP_MAX_GROUP = 128;

// A line of work (paged_schedule.h) with the scratch of its units' parts.
struct PagedLineArgs {
  PagedLine line;     // ctas == 0: nothing can be on it
  int box_log2;       // rows of a K or V box
  uint32_t *arrived;  // [AP_LEVELS][line.ctas][8]: parts of a group that are parked; zero when they are first used
  // parked parts, [2 * line.ctas, and line.ctas more of few rows][rows of a unit]: unnormalised o, DH floats in whole lines, and
  // (m, l), its reference point and sum
  float *parts;
  float2 *parts_ml;
  PagedDiv by_ctas[AP_SHARES];  // by the CTAs that are this line's where both have work, by paged_share
};

struct PagedAttnArgs {
  const char *q, *k, *v;
  char *o;
  long long q_h, q_t, o_h, o_t;                  // byte strides: head, token
  long long kp_p, kp_h, kp_s, vp_p, vp_h, vp_s;  // byte strides: page, head, slot
  int nh, dh;
  float scale_log2;  // scale * log2(e): the softmax runs in powers of two
  int odd_scale;     // scale <= 0
  int per_tile;      // tokens of a tile: 128 / query heads of a kv head
  unsigned long long patience;  // ns that a warp waits for the other parts of a unit of more than two
  PagedBatch batch;
  PagedLineArgs few, tile;
};

// Tensor maps: K and V of the whole cache, boxes of 64 columns x 2^box_log2 slots of one head of one page; the queries, boxes of 64
// columns x the heads of a group x the tokens of a tile.
struct PagedAttnMaps {
  CUtensorMap few_k, few_v, tile_q, tile_k, tile_v;
};
// Launches the kernel for few rows alone (tiles == false) or for both, of 8 or 16 few rows.  `prepared`: the handle's.
int attention_paged_run_f16(const PagedAttnMaps &maps, const PagedAttnArgs &a, int few_rows, bool tiles, std::atomic<unsigned> &prepared, cudaStream_t s);
int attention_paged_run_bf16(const PagedAttnMaps &maps, const PagedAttnArgs &a, int few_rows, bool tiles, std::atomic<unsigned> &prepared, cudaStream_t s);

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

// What of the two lines is this CTA's, by its warps `few_finder` and `tile_finder` (TILES), for all behind the next barrier.  All sequences' points are added up, then the sequence that the share
// begins in is looked for.  Up to 32 sequences are the finders' alone; of more, every warp of the CTA adds up an even part
// first and a finder looks for its sequence in one of the parts: all warps call, and meet once.  (One warp alone took a round trip
// to memory per 32 sequences, twice: 30 us of 2048 decoding requests' 116.)  CTA 0 looks for what is wrong with the batch.
//
// Where neither line is empty the two split the CTAs, and the SMs with them.  One after the other, the first would leave the
// tensor cores idle and the second the memory; and of the 148 SMs 96 are enough to read as fast as all (72: 89 %, 48: 63 %).  The
// split makes both take as long, by what a key costs an SM: 4 dh bytes at 68 GB/s, or 4 dh flops for each of 256 rows at
// 7 TFLOP/s, 2.5 times as long (a chunk of 487 tokens beside 31 single ones over up to 2900 keys: 64 us, 86 one after the other).
// Short sequences are bound by their number, not by the memory, and gain nothing from fewer SMs (512 single tokens over 100
// keys beside eight prompts of 700 tokens: 72 us, 66 one after the other): then only a small share of the work runs beside the
// other's (64 of them: 47 us, 53 one after the other).
struct PagedShare {
  int cta;  // place on the line, -1: nothing there
  int total;
  int ctas;  // that have a part of it
  PagedDiv by_ctas;
  PagedWalk walk;
};
__device__ __forceinline__ PagedLine paged_shared_line(const PagedLine &l, const PagedShare &s) {
  PagedLine mine = l;
  mine.ctas = s.ctas;
  mine.by_ctas = s.by_ctas;
  return mine;
}

template <int WARPS, bool TILES>
__device__ __forceinline__ void paged_locate(const PagedAttnArgs &a, int warp, int few_finder, int tile_finder, PagedShare (&shares)[2]) {
  static_assert(WARPS <= 32, "a lane per part");
  __shared__ int parts[3][WARPS];  // points of the lines (-1: too many), sequences of few rows
  const PagedBatch &b = a.batch;
  const int lane = threadIdx.x & 31, nkvh = a.few.line.nkvh;
  const bool few = !TILES || warp == few_finder, finder = warp == few_finder || (TILES && warp == tile_finder), report = blockIdx.x == 0;
  PagedShare &mine = shares[few ? 0 : 1];
  if (finder && lane == 0) mine.cta = -1;
  const bool together = b.nseq > 32;
  if (!together && !finder) return;
  const int part = together ? (b.nseq + WARPS * 32 - 1) / (WARPS * 32) * 32 : 32;
  int i0 = together ? warp * part : 0, end = min(b.nseq, i0 + part);
  long long few_sum = 0, tile_sum = 0;
  int few_seqs = 0, lo = 0, hi = 0, cta = 0, total = 0, before = 0;
  PagedLine line = few ? a.few.line : a.tile.line;
  auto all_lanes = [](long long x) -> long long {  // the sum of non-negative numbers
    x = min(x, 1ll << 40);  // far more than a line holds; the halves of 32 such sums add up in 32 bits
    return (long long)__reduce_add_sync(0xffffffffu, (unsigned)(x & 0xffffff)) + ((long long)__reduce_add_sync(0xffffffffu, (unsigned)(x >> 24)) << 24);
  };
  auto fits = [](long long x) -> int { return x <= 0x7fffffff ? (int)x : -1; };
  bool looking = false, picking = false;  // for a sequence, for a part; both passes run through one copy of the code
#pragma unroll 1
  while (true) {
    const int i = i0 + lane;
    long long few_cost = 0, tile_cost = 0;
    if (i < end) {
      const PagedSeq s = paged_seq(b, i, report && !looking);
      few_cost = (long long)paged_span(a.few.line, s).head * nkvh;
      if (TILES) tile_cost = (long long)paged_span(a.tile.line, s).head * nkvh;
    }
    int cost = (int)(few ? few_cost : tile_cost);
    i0 += 32;
    if (!looking) {
      few_sum += few_cost;
      if (TILES) {
        tile_sum += tile_cost;
        few_seqs += few_cost > 0;
      }
      if (i0 < end) continue;
      few_sum = all_lanes(few_sum);
      if (TILES) {
        tile_sum = all_lanes(tile_sum);
        few_seqs = __reduce_add_sync(0xffffffffu, few_seqs);
      }
      if (together) {
        if (lane == 0) {
          parts[0][warp] = fits(few_sum);
          parts[1][warp] = fits(tile_sum);
          parts[2][warp] = few_seqs;
        }
        __syncthreads();
        if (!finder) return;
        const int f = lane < WARPS ? parts[0][lane] : 0, t = lane < WARPS ? parts[1][lane] : 0;
        few_sum = all_lanes(f < 0 ? 1ll << 40 : f);
        if (TILES) {
          tile_sum = all_lanes(t < 0 ? 1ll << 40 : t);
          few_seqs = __reduce_add_sync(0xffffffffu, lane < WARPS ? parts[2][lane] : 0);
        }
        cost = few ? f : t;
      }
      // sequences that share rows (seq_start falls) can put more on a line than the host allowed for: nothing is done then
      const int few_total = max(0, fits(few_sum)), tile_total = max(0, fits(tile_sum));
      if (report && few && (few_total != few_sum || tile_total != tile_sum) && lane == 0) atomicCAS(b.status, 0, OPS_PAGED_BAD_ROWS);
      total = few ? few_total : tile_total;
      cta = blockIdx.x;
      if (TILES && few_total > 0 && tile_total > 0) {
        const float few_keys = (float)few_total * (float)(1u << a.few.line.shift);
        const float tile_keys = 2.5f * (float)tile_total * (float)(1u << a.tile.line.shift);  // in what a key of few rows costs
        if (few_keys >= 768.f * (float)few_seqs * (float)nkvh || 13.f * few_keys <= 3.f * tile_keys) {  // 640 keys a unit and more, or 3 / 16 of the work
          const int k = min(max(__float2int_rn(AP_SHARES * few_keys / (few_keys + tile_keys)), 1), AP_SHARES * 3 / 4);
          const int few_ctas = paged_share(a.few.line.ctas, k);
          line.ctas = few ? few_ctas : a.tile.line.ctas - few_ctas;
          line.by_ctas = few ? a.few.by_ctas[k] : a.tile.by_ctas[k];
          if (!few) cta -= few_ctas;
        }
      }
      if (cta < 0 || cta >= line.ctas) return;
      lo = paged_cut(line, total, cta);
      hi = paged_cut(line, total, cta + 1);
      if (lo >= hi) return;
      looking = true;
      picking = together;
    }
    int upto = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned here = __ballot_sync(0xffffffffu, before + upto - cost <= lo && lo < before + upto);
    if (here) {
      const int at = __ffs(here) - 1;
      before += __shfl_sync(0xffffffffu, upto - cost, at);
      if (!picking) {
        if (lane == 0) {
          mine.cta = cta;
          mine.total = total;
          mine.ctas = line.ctas;
          mine.by_ctas = line.by_ctas;
          mine.walk = {i0 - 32 + at, before, lo, hi};
        }
        return;
      }
      picking = false;
      i0 = at * part;
      end = min(b.nseq, i0 + part);
      continue;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// By one thread.  Between two chunks far apart in a batch there may be thousands of single tokens or idle sequences, which have
// nothing on the line: the thread looks at 16 of them a round trip to memory, 20 ns each (one a round trip, 140 ns each: the launch of
// two chunks with 4000 single tokens between them 631 us, now 243, 88 with the chunks side by side; with 4000 idle sequences 550,
// 106 and 27).  Passing over whole runs that paged_locate has found empty, or a warp that looks at 32, comes to 105 to 117 us, but
// as code in every launch costs one token 0.1 to 0.3 us and a chunk beside single tokens 1.5 of 63.
__device__ __forceinline__ PagedPiece paged_step(const PagedBatch &b, const PagedLine &l, PagedWalk &w) {
  return paged_next(l, b.nseq, w, [&](int i) { return paged_seq(b, i, false); }, [&](int seq) {
    constexpr int AT_ONCE = 16;
#pragma unroll 1
    for (; seq + AT_ONCE <= b.nseq; seq += AT_ONCE) {
      uint32_t start[AT_ONCE + 1];
#pragma unroll
      for (int e = 0; e <= AT_ONCE; ++e) start[e] = min(b.start[seq + e], (uint32_t)b.nt);
      int first = AT_ONCE;
#pragma unroll
      for (int e = AT_ONCE - 1; e >= 0; --e)
        if (paged_rows_fit(l, start[e], start[e + 1])) first = e;
      if (first < AT_ONCE) return seq + first;
    }
    return seq;
  });
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
// may come, the other waits for all of its results.  (Here: the kernel that clears the counters, the one that uses them.)
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
