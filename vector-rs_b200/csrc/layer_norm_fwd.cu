// layer_norm_fwd.cu -- y = (x - mean) * rstd * weight + bias over rows, with
// mean and rstd = 1 / sqrt(var + eps) kept in 32 bits for the backward pass.
//
// Bound by memory: 2 d elements a row. The row stays in registers between the
// two sums (mean first, then the squares of x - mean: one pass of
// sum-of-squares would lose the variance of rows whose mean is large).
#include <atomic>

#include "layer_norm.cuh"

namespace vrs {
namespace ops {
namespace {

// Elements a thread holds: with 32 a warp covers 1,024 elements with no
// barrier at all.
constexpr int kE = 32;

template <class T, class P, int VEC, int TPR, bool CL>
__global__ void __launch_bounds__(kLnThreads) ln_fwd_kernel(const LnArgs a) {
  constexpr int NV = kE / VEC, GROUPS = kLnThreads / TPR;
  using Red = LnReduce<TPR, CL, 1>;
  __shared__ typename Red::Smem s_red;
  int tt = threadIdx.x % TPR, TT = TPR;
  int64_t first = blockIdx.x, step = gridDim.x;
  if constexpr (CL) {
    auto cluster = cooperative_groups::this_cluster();
    TT = TPR * (int)cluster.num_blocks();
    tt += TPR * (int)cluster.block_rank();
    first /= cluster.num_blocks();
    step /= cluster.num_blocks();
  }
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  const P* w = (const P*)a.weight;
  const P* b = (const P*)a.bias;
  const float inv_d = 1.0f / (float)a.d;
  int slot = 0;
  // Every thread of a block takes the same number of turns (the barriers
  // inside the reductions); a group past the last row computes on zeros.
  for (int64_t r0 = first * GROUPS; r0 < a.rows; r0 += step * GROUPS) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool have = row < a.rows;
    Pack<T, VEC> k[NV];
    float v[kE];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (i * TT + tt) * VEC;
      if (have && c < a.d) {
        k[i] = load_pack<T, VEC>(x + row * a.xs + c);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) k[i].v[j] = from_f32<T>(0.0f);
      }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < VEC; j++) sum += v[i * VEC + j] = to_f32(k[i].v[j]);
    Red::run(&sum, &s_red, slot);
    slot ^= 1;
    const float mean = sum * inv_d;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const bool in = (i * TT + tt) * VEC < a.d;
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        v[i * VEC + j] -= mean;
        if (in) sq = fmaf(v[i * VEC + j], v[i * VEC + j], sq);
      }
    }
    Red::run(&sq, &s_red, slot);
    slot ^= 1;
    const float rstd = 1.0f / sqrtf(fmaf(sq, inv_d, a.eps));
    if (!have) continue;
    if (tt == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (i * TT + tt) * VEC;
      if (c >= a.d) continue;
      float o[VEC], f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) o[j] = v[i * VEC + j] * rstd;
      if (w) {
        load_params<P, VEC>(w + c, f);
#pragma unroll
        for (int j = 0; j < VEC; j++) o[j] *= f[j];
      }
      if (b) {
        load_params<P, VEC>(b + c, f);
#pragma unroll
        for (int j = 0; j < VEC; j++) o[j] += f[j];
      }
      store_pack<T, VEC>(y + row * a.ys + c, o);
    }
  }
  // A block must not leave while another still writes its shared memory.
  if constexpr (CL) cooperative_groups::this_cluster().sync();
}

template <class T, class P, int VEC, int TPR, bool CL>
struct FwdKernel {
  static auto get() { return &ln_fwd_kernel<T, P, VEC, TPR, CL>; }
};

}  // namespace

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

int ln_check(const char* who, int64_t rows, int64_t d, int32_t dtype, int32_t param_dtype) {
  if (dtype < VRS_F32 || dtype > VRS_BF16) return invalid(std::string(who) + ": dtype must be f32, f16 or bf16");
  if (param_dtype != dtype && param_dtype != VRS_F32)
    return invalid(std::string(who) + ": parameters are in the rows' type or f32");
  if (rows < 0) return invalid(std::string(who) + ": negative row count");
  if (d < 1 || d > kLnMaxD) return invalid(std::string(who) + ": d must be in 1.." + std::to_string(kLnMaxD));
  return VRS_OK;
}

}  // namespace ops
}  // namespace vrs

extern "C" int vrs_layer_norm_forward(const void* x, int64_t x_stride, int64_t rows, int64_t d, int32_t dtype,
                                      const void* weight, const void* bias, int32_t param_dtype, float eps, void* y,
                                      int64_t y_stride, float* mean, float* rstd, void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  VRS_TRY(ln_check("vrs_layer_norm_forward", rows, d, dtype, param_dtype));
  if (!(eps >= 0.0f)) return invalid("vrs_layer_norm_forward: eps must be at least 0");
  if (rows == 0) return VRS_OK;
  if (!x || !y) return invalid("vrs_layer_norm_forward: null x or y");
  if (rows > 1 && (x_stride < d || y_stride < d))
    return invalid("vrs_layer_norm_forward: row strides must be at least d");
  LnArgs a{};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = rows;
  a.xs = x_stride;
  a.ys = y_stride;
  a.d = (int)d;
  a.eps = eps;
  const int vec = 16 / dtype_bytes(dtype);
  const bool can_vec = d % vec == 0 && (rows == 1 || (x_stride % vec == 0 && y_stride % vec == 0)) && aligned16(x) &&
                       aligned16(y) && aligned16(weight) && aligned16(bias);
  int sms = 0;
  VRS_TRY(sm_count(&sms));
  const LnPlan p = ln_plan(rows, (int)d, kE, vec, can_vec, sms, 6);
  cudaStream_t s = (cudaStream_t)cuda_stream;
  ProfToken t = prof_begin("layer_norm_forward", s);
  const int st = ln_dispatch<FwdKernel>(dtype, param_dtype, a, p, s);
  prof_end(t, s);
  return st;
}
