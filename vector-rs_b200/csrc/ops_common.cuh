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

__device__ __forceinline__ void round_pair(f16* o, float lo, float hi) {
  *reinterpret_cast<__half2*>(o) = __floats2half2_rn(lo, hi);
}
__device__ __forceinline__ void round_pair(bf16* o, float lo, float hi) {
  *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(lo, hi);
}
__device__ __forceinline__ void round_pair(float* o, float lo, float hi) {
  o[0] = lo;
  o[1] = hi;
}

template <class T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float* v) {
  Pack<T, VEC> o;
  if constexpr (VEC == 1) {
    o.v[0] = from_f32<T>(v[0]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) round_pair(o.v + j, v[j], v[j + 1]);
  }
  *reinterpret_cast<Pack<T, VEC>*>(p) = o;
}

// ---- pairs of floats: sm_100 multiplies and adds two at once (f32x2), which
// halves the instructions of kernels that are short of issue slots.
struct F2 {
  unsigned long long u;
};
__device__ __forceinline__ F2 pack_f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.u) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 pack_f2(float v) { return pack_f2(v, v); }
__device__ __forceinline__ void unpack_f2(F2 a, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.u));
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ float sum_f2(F2 a) {
  float lo, hi;
  unpack_f2(a, lo, hi);
  return lo + hi;
}

// Two neighbouring elements as floats (a bf16 is the upper half of a float).
__device__ __forceinline__ F2 pair_of(const float* p) { return pack_f2(p[0], p[1]); }
__device__ __forceinline__ F2 pair_of(const f16* p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
  return pack_f2(f.x, f.y);
}
__device__ __forceinline__ F2 pair_of(const bf16* p) {
  const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
  return pack_f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// E elements of a row or of a parameter array in a thread's registers, in
// their own type, as NV accesses of VEC.
template <class T, int E, int VEC>
struct Held {
  static constexpr int NV = E / VEC;
  static_assert(VEC * sizeof(T) <= 16 || VEC * sizeof(T) == 32, "one or two 16-byte accesses");
  Pack<T, VEC> k[NV];
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < VEC; j++) k[i].v[j] = from_f32<T>(f);
  }
  // 32-bit parameters beside 16-bit rows: a pack of 8 takes two accesses.
  __device__ __forceinline__ void load(int i, const T* p) {
    constexpr int H = sizeof(T) * VEC > 16 ? 16 / (int)sizeof(T) : VEC;
#pragma unroll
    for (int h = 0; h < VEC / H; h++) {
      const Pack<T, H> q = load_pack<T, H>(p + h * H);
#pragma unroll
      for (int j = 0; j < H; j++) k[i].v[h * H + j] = q.v[j];
    }
  }
  // Elements 2q and 2q + 1 as floats.
  __device__ __forceinline__ F2 pair(int q) const {
    if constexpr (VEC > 1)
      return pair_of(&k[2 * q / VEC].v[2 * q % VEC]);
    else
      return pack_f2(to_f32(k[2 * q].v[0]), to_f32(k[2 * q + 1].v[0]));
  }
};

// Stores a pair-wise row: VEC elements at access i.
template <class T, int VEC, int E>
__device__ __forceinline__ void store_held(T* p, const F2 (&v)[E / 2], int i) {
  float f[VEC];
  if constexpr (VEC == 1) {
    float lo, hi;
    unpack_f2(v[i / 2], lo, hi);
    f[0] = i & 1 ? hi : lo;
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) unpack_f2(v[(i * VEC + j) / 2], f[j], f[j + 1]);
  }
  store_pack<T, VEC>(p, f);
}

// ---- dependent launches. A kernel started by launch_after may begin while the
// one before it on the stream ends: it waits (grid_wait) before it touches
// memory, for that kernel and, since every kernel here does so, for all before
// it. grid_launch lets the next one begin once all blocks have come so far.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... KA, class... A>
int launch_after(void (*kernel)(KA...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  VRS_CUDA(cudaLaunchKernelEx(&cfg, kernel, KA(args)...));
  return VRS_OK;
}

inline int dtype_bytes(int dtype) { return dtype == VRS_F32 ? 4 : 2; }

inline int invalid(const std::string& m) {
  set_error(VRS_ERR_INVALID_CONFIG, m);
  return VRS_ERR_INVALID_CONFIG;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// SMs of the current device (148 on B200), read once per device.
int sm_count(int* out);

// The word that a device wait which gave up writes: host memory that the
// device sees, so a later call reads it without waiting for anything. An
// earlier call's gives VRS_ERR_TIMEOUT once, here or from vrs_operators_status.
int error_word(int** out);

}  // namespace ops
}  // namespace vrs
