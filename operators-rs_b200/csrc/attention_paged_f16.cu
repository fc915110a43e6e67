// attention_paged_f16.cu — the kernels of attention_paged for f16 (a file per type: they take a minute to compile).
#include "attention_paged_kernel.cuh"

namespace ops {

int attention_paged_run_f16(const PagedAttnMaps &maps, const PagedAttnArgs &a, int few_rows, bool tiles, std::atomic<unsigned> &prepared, cudaStream_t s) {
  return paged_kernel_launch<false>(maps, a, few_rows, tiles, prepared, s);
}

}  // namespace ops
