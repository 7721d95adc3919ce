// ops_common.cuh -- element types, vector access and argument checks shared by
// the training operators (layer_norm_*.cu, linear_ce*.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vrs_internal.cuh"

namespace vrs {
namespace ops {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }

// Round to nearest even, the one rounding of a result kept in 16 bits.
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }

// VEC consecutive elements moved by one load or store (16 bytes, or one element).
template <class T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T v[VEC];
};

template <class T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

template <class T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float* v) {
  Pack<T, VEC> o;
#pragma unroll
  for (int j = 0; j < VEC; j++) o.v[j] = from_f32<T>(v[j]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = o;
}

// VEC parameters (weights or biases) in 32 bits; a 32-bit parameter array
// beside 16-bit rows takes two 16-byte loads.
template <class P, int VEC>
__device__ __forceinline__ void load_params(const P* p, float* out) {
  if constexpr (sizeof(P) * VEC > 16) {
    constexpr int H = 16 / sizeof(P);
#pragma unroll
    for (int h = 0; h < VEC / H; h++) {
      const Pack<P, H> k = load_pack<P, H>(p + h * H);
#pragma unroll
      for (int j = 0; j < H; j++) out[h * H + j] = to_f32(k.v[j]);
    }
  } else {
    const Pack<P, VEC> k = load_pack<P, VEC>(p);
#pragma unroll
    for (int j = 0; j < VEC; j++) out[j] = to_f32(k.v[j]);
  }
}

inline int dtype_bytes(int dtype) { return dtype == VRS_F32 ? 4 : 2; }

inline int invalid(const std::string& m) {
  set_error(VRS_ERR_INVALID_CONFIG, m);
  return VRS_ERR_INVALID_CONFIG;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// SMs of the current device (148 on B200), read once per device.
int sm_count(int* out);

}  // namespace ops
}  // namespace vrs
