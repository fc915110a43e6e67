// paged.cu — the status words of the paged operators' handles.
#include "paged.h"

namespace ops {

int paged_create(PagedHandle *h, int device) {
  h->status = nullptr;
  OPS_TRY(init_base(&h->base, device));
  DeviceGuard guard(device);
  if (cudaMalloc(&h->status, 2 * sizeof(int)) != cudaSuccess || zero_words(h->status, 2 * sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    if (h->status) cudaFree(h->status);
    return fail(OPS_EXECUTION_FAILED, "cannot allocate the status words");
  }
  return OPS_OK;
}

void paged_destroy(PagedHandle *h) {
  if (h->status) cudaFree(h->status);
}

int paged_status(const PagedHandle *h) {
  DeviceGuard guard(h->base.device);
  int v[2];
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpy(v, h->status, sizeof(v), cudaMemcpyDeviceToHost) != cudaSuccess) return -1;
  return v[1] ? v[1] : v[0];
}

int paged_status_reset(PagedHandle *h) {
  DeviceGuard guard(h->base.device);
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = zero_words(h->status, 2 * sizeof(int));
  if (e != cudaSuccess) return fail(OPS_EXECUTION_FAILED, "status reset: %s", cudaGetErrorString(e));
  return OPS_OK;
}

}  // namespace ops
