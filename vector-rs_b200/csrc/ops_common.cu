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

namespace {

std::mutex g_word_lock;
int* g_word = nullptr;  // taken by the first call

// What a wait left in the word, once. (With the lock held.)
int word_status() {
  const int code = g_word ? *(volatile int*)g_word : 0;
  if (!code) return VRS_OK;
  *(volatile int*)g_word = 0;
  set_error(VRS_ERR_TIMEOUT, "training operators: a device wait of an earlier call gave up (stage code " +
                                 std::to_string(code) + "); its results are not valid");
  return VRS_ERR_TIMEOUT;
}

}  // namespace

int error_word(int** out) {
  std::lock_guard<std::mutex> g(g_word_lock);
  if (!g_word) {
    void* p = nullptr;
    VRS_CUDA(cudaHostAlloc(&p, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped));
    g_word = static_cast<int*>(p);
    *g_word = 0;
  }
  VRS_TRY(word_status());
  *out = g_word;
  return VRS_OK;
}

}  // namespace ops
}  // namespace vrs

extern "C" int vrs_operators_status(void) {
  std::lock_guard<std::mutex> g(vrs::ops::g_word_lock);
  return vrs::ops::word_status();
}
