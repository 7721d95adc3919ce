// layer_norm.cuh -- what the layer norm's forward and backward kernels share:
// the launch plan, the split of a row over threads, and its reductions.
//
// A row of d elements is held in registers by TPR threads (32 to 256) of a
// 256-thread block, or by a cluster of 2 to 8 blocks, E elements a thread, so
// that it is read from memory once. Thread tt of a row's TT threads holds the
// vectors i * TT + tt: neighbouring threads read neighbouring 16 bytes. Rows
// that 16-byte accesses cannot reach (odd widths, strides or addresses) take
// the same kernels with one element per access.
#pragma once
#include <cooperative_groups.h>

#include "ops_common.cuh"

namespace vrs {
namespace ops {

constexpr int kLnThreads = 256;
constexpr int kLnMaxCluster = 8;
constexpr int64_t kLnMaxD = 32768;

struct LnArgs {
  const void* x;
  const void* dy;      // backward
  const void* weight;  // nullable: ones
  const void* bias;    // forward, nullable: zeros
  void* y;             // forward: y; backward: dx
  const float* mean_in;
  const float* rstd_in;
  float* mean;
  float* rstd;
  float* partial;      // backward: [row blocks][2][d], null without parameter gradients
  int64_t rows;
  int64_t xs, dys, ys;  // row strides in elements
  int d;
  float eps;
};

struct LnPlan {
  int tpr;      // threads of a row within a block (32..256)
  int cluster;  // blocks of a row (1: none)
  bool vec;     // 16-byte accesses
  int blocks;   // grid, in clusters
};

// E: elements a thread holds. The fewest threads that hold a row; a row wider
// than one block takes a cluster, and so do rows so few that blocks alone
// would leave most SMs idle (each thread still has at least one access).
inline LnPlan ln_plan(int64_t rows, int d, int e, int vec, bool can_vec, int sms, int blocks_per_sm) {
  LnPlan p{};
  p.vec = can_vec;
  const int step = can_vec ? vec : 1;
  p.tpr = 32;
  while (p.tpr < kLnThreads && p.tpr * e < d) p.tpr *= 2;
  p.cluster = 1;
  if (p.tpr == kLnThreads) {
    while (p.cluster < kLnMaxCluster && p.cluster * kLnThreads * e < d) p.cluster *= 2;
    while (p.cluster < kLnMaxCluster && rows * p.cluster * 2 <= sms && (int64_t)p.cluster * 2 * kLnThreads * step <= d)
      p.cluster *= 2;
  }
  const int groups = kLnThreads / p.tpr;
  const int64_t need = (rows + groups - 1) / groups;
  const int64_t most = (int64_t)sms * blocks_per_sm / p.cluster;
  p.blocks = (int)(need < most ? need : most);
  if (p.blocks < 1) p.blocks = 1;
  return p;
}

// Sums of N values over the threads of a row, the same bits in all of them.
// `slot` alternates between two buffers, so one barrier a reduction suffices:
// a buffer is written again only after the next reduction's barrier.
template <int TPR, bool CL, int N>
struct LnReduce {
  static constexpr int kWarps = kLnThreads / 32;
  struct Smem {
    float warp[2][kWarps][N];
    float cta[2][kLnMaxCluster][N];
  };
  __device__ static __forceinline__ void run(float* v, Smem* s, int slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int n = 0; n < N; n++) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    if constexpr (TPR > 32) {
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
      if (lane == 0)
#pragma unroll
        for (int n = 0; n < N; n++) s->warp[slot][warp][n] = v[n];
      __syncthreads();
      constexpr int W = TPR / 32;
      const int w0 = warp / W * W;
#pragma unroll
      for (int n = 0; n < N; n++) v[n] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; w++)
#pragma unroll
        for (int n = 0; n < N; n++) v[n] += s->warp[slot][w0 + w][n];
    }
    if constexpr (CL) {
      auto cluster = cooperative_groups::this_cluster();
      const int c = (int)cluster.num_blocks(), r = (int)cluster.block_rank();
      if ((int)threadIdx.x < c) {
        float* to = cluster.map_shared_rank(&s->cta[slot][r][0], threadIdx.x);
#pragma unroll
        for (int n = 0; n < N; n++) to[n] = v[n];
      }
      cluster.sync();
#pragma unroll
      for (int n = 0; n < N; n++) v[n] = 0.0f;
      for (int b = 0; b < c; b++)
#pragma unroll
        for (int n = 0; n < N; n++) v[n] += s->cta[slot][b][n];
    }
  }
};

template <class K>
int ln_launch(K kernel, const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.blocks * p.cluster));
  cfg.blockDim = dim3(kLnThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  if (p.cluster > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  VRS_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  count_launch();
  return VRS_OK;
}

// The instantiation for a plan: K<T, P, VEC, TPR, CL>::get().
template <template <class, class, int, int, bool> class K, class T, class P, int VEC>
int ln_dispatch_tpr(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  if (p.cluster > 1) return ln_launch(K<T, P, VEC, kLnThreads, true>::get(), a, p, s);
  switch (p.tpr) {
    case 32: return ln_launch(K<T, P, VEC, 32, false>::get(), a, p, s);
    case 64: return ln_launch(K<T, P, VEC, 64, false>::get(), a, p, s);
    case 128: return ln_launch(K<T, P, VEC, 128, false>::get(), a, p, s);
    default: return ln_launch(K<T, P, VEC, 256, false>::get(), a, p, s);
  }
}

template <template <class, class, int, int, bool> class K, class T, class P>
int ln_dispatch_vec(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  return p.vec ? ln_dispatch_tpr<K, T, P, 16 / (int)sizeof(T)>(a, p, s) : ln_dispatch_tpr<K, T, P, 1>(a, p, s);
}

template <template <class, class, int, int, bool> class K>
int ln_dispatch(int dtype, int param_dtype, const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  switch (dtype) {
    case VRS_F32: return ln_dispatch_vec<K, float, float>(a, p, s);
    case VRS_F16:
      return param_dtype == VRS_F32 ? ln_dispatch_vec<K, f16, float>(a, p, s) : ln_dispatch_vec<K, f16, f16>(a, p, s);
    default:
      return param_dtype == VRS_F32 ? ln_dispatch_vec<K, bf16, float>(a, p, s)
                                    : ln_dispatch_vec<K, bf16, bf16>(a, p, s);
  }
}

int ln_check(const char* who, int64_t rows, int64_t d, int32_t dtype, int32_t param_dtype);

}  // namespace ops
}  // namespace vrs
