// attention_paged_bf16.cu — the kernels of attention_paged for bf16 (a file per type: they take a minute to compile).
#include "attention_paged_kernel.cuh"

namespace ops {

int attention_paged_run_bf16(const PagedAttnMaps &maps, const PagedAttnArgs &a, int few_rows, bool tiles, std::atomic<unsigned> &prepared, cudaStream_t s) {
  return paged_kernel_launch<true>(maps, a, few_rows, tiles, prepared, s);
}

}  // namespace ops
