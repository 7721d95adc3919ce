// ops_common.cu -- what the training operators' host code shares.
#include <atomic>
#include <mutex>

#include "ops_common.cuh"

namespace vrs {
namespace ops {

int sm_count(int* out) {
  static std::atomic<int> cached[128];  // zero: not read yet
  int dev = 0;
  VRS_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 128 || !cached[dev]) {
    int n = 0;
    VRS_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 0 || dev >= 128) {
      *out = n;
      return VRS_OK;
    }
    cached[dev] = n;
  }
  *out = cached[dev];
  return VRS_OK;
}

int error_word(int** out) {
  static std::mutex mu;
  static int* word = nullptr;
  std::lock_guard<std::mutex> g(mu);
  if (!word) {
    void* p = nullptr;
    VRS_CUDA(cudaHostAlloc(&p, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped));
    word = static_cast<int*>(p);
    *word = 0;
  }
  const int code = *(volatile int*)word;
  if (code) {
    *(volatile int*)word = 0;
    set_error(VRS_ERR_TIMEOUT, "training operators: a device wait of an earlier call gave up (stage code " +
                                   std::to_string(code) + "); its results are not valid");
    return VRS_ERR_TIMEOUT;
  }
  *out = word;
  return VRS_OK;
}

}  // namespace ops
}  // namespace vrs
