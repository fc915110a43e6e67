// attention_paged_kernel.cuh — the kernel of attention_paged: a CTA's share of the line of few rows, then, or instead, of the line of
// tiles (paged_locate says which), in one launch.  (As two launches beside each other a prompt waited 3 us for an idle one, and a
// launch costs the host 2.5 us.)  Where max_seq leaves no work for tiles, a kernel without them.
#pragma once
#include "attention_paged_few.cuh"
#include "attention_paged_tile.cuh"

namespace ops {

template <int DH, int NR, bool TILES> constexpr int paged_kernel_bytes() {
  return TILES && TileSmem<DH>::BYTES > FewSmem<DH, NR>::BYTES ? TileSmem<DH>::BYTES : FewSmem<DH, NR>::BYTES;
}

template <int DH, bool BF, int NR, bool TILES>
__global__ void __launch_bounds__(TILES ? TL_THREADS : FEW_THREADS, 1)
    attention_paged_kernel(const __grid_constant__ PagedAttnMaps maps, const __grid_constant__ PagedAttnArgs a) {
  constexpr int THREADS = TILES ? TL_THREADS : FEW_THREADS, FEW_FINDER = FEW_CONSUMERS + FEW_PRODUCERS, TILE_FINDER = 3;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *base_ptr = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  __shared__ FewShared<DH, NR> few_sh;
  __shared__ TileShared<DH> tile_sh;
  __shared__ PagedShare shares[2];
  __shared__ int gave_up;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  paged_locate<THREADS / 32, TILES>(a, warp, FEW_FINDER, TILE_FINDER, shares);
  if (threadIdx.x == 0) {
    gave_up = 0;
    few_init(few_sh);
    if (TILES) tile_init(tile_sh);
    fence_barrier_init();
  }
  if (warp == 4 && lane == 0) {
    if (!TILES || a.few.line.ctas) {
      tma_prefetch_desc(&maps.few_k);
      tma_prefetch_desc(&maps.few_v);
    }
    if (TILES) {
      tma_prefetch_desc(&maps.tile_q);
      tma_prefetch_desc(&maps.tile_k);
      tma_prefetch_desc(&maps.tile_v);
    }
  }
  if (TILES && warp == 1) {
    tmem_alloc(smem_u32(&tile_sh.tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  bool ok = true;
  if (shares[0].cta >= 0) {
    ok = few_rows<DH, BF, NR>(maps.few_k, maps.few_v, a, base_ptr, few_sh, shares[0]);
    if (!ok) gave_up = 1;
    if (TILES) fence_proxy_async();  // what was written here is overwritten through the async proxy
    __syncthreads();
    ok = !*(volatile int *)&gave_up;
  }
  if (TILES) {
    if (shares[1].cta >= 0 && ok) {
      ok = tiles<DH, BF>(maps.tile_q, maps.tile_k, maps.tile_v, a, base_ptr, tile_sh, shares[1]);
      if (!ok) gave_up = 1;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  pdl_wait_for_front();  // (no launch ends in front of the one it started beside; who uses the counters has waited for them to be cleared)
  if (*(volatile int *)&gave_up) __nanosleep(1000000);  // a wait ran out: let stray copies land before the CTA goes away
  if (TILES && threadIdx.x >> 5 == 1) tmem_dealloc(tile_sh.tmem, 512);
}

template <int DH, bool BF, int NR, bool TILES>
static int paged_kernel_launch(const PagedAttnMaps &maps, const PagedAttnArgs &a, std::atomic<unsigned> &prepared, cudaStream_t s) {
  const int ctas = a.few.line.ctas > a.tile.line.ctas ? a.few.line.ctas : a.tile.line.ctas;
  return ap_launch_beside("attention_paged", prepared, 1u << ((DH == 128) * 8 + BF * 4 + TILES * 2 + NR - 1), attention_paged_kernel<DH, BF, NR, TILES>, ctas,
                          TILES ? TL_THREADS : FEW_THREADS, paged_kernel_bytes<DH, NR, TILES>(), s, maps, a);
}
template <int DH, bool BF>
static int paged_kernel_launch(const PagedAttnMaps &maps, const PagedAttnArgs &a, int few_rows, bool tiles, std::atomic<unsigned> &prepared, cudaStream_t s) {
  if (few_rows == 8) return tiles ? paged_kernel_launch<DH, BF, 1, true>(maps, a, prepared, s) : paged_kernel_launch<DH, BF, 1, false>(maps, a, prepared, s);
  return tiles ? paged_kernel_launch<DH, BF, 2, true>(maps, a, prepared, s) : paged_kernel_launch<DH, BF, 2, false>(maps, a, prepared, s);
}
template <bool BF>
static int paged_kernel_launch(const PagedAttnMaps &maps, const PagedAttnArgs &a, int few_rows, bool tiles, std::atomic<unsigned> &prepared, cudaStream_t s) {
  return a.dh <= 64 ? paged_kernel_launch<64, BF>(maps, a, few_rows, tiles, prepared, s) : paged_kernel_launch<128, BF>(maps, a, few_rows, tiles, prepared, s);
}

}  // namespace ops
