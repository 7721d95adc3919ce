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

#include <atomic>

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
  float* partial;      // backward: [row blocks][2][d], null where it is not needed
  void* dweight;       // backward: written by column blocks (few rows), nullable
  void* dbias;
  int col_blocks;      // backward: blocks of the grid that sum columns
  int64_t rows;
  int64_t xs, dys, ys;  // row strides in elements
  int d;
  float eps;
};

struct LnPlan {
  int tpr;      // threads of a row within a block (32..256)
  int cluster;  // blocks of a row (1: none)
  bool vec;     // 16-byte accesses
  bool wide;    // more elements a thread
  int blocks;   // grid, in clusters
};

// A thread holds `narrow` elements of a row of up to one block of them, else
// `wide`, of rows_narrow or rows_wide rows at a time. The fewest threads that hold a row; a row wider than one block takes
// a cluster, and so do rows so few that blocks alone would leave most SMs idle
// (each thread still has at least one access).
inline LnPlan ln_plan(int64_t rows, int d, int narrow, int wide, int rows_narrow, int rows_wide, int vec,
                      bool can_vec, int sms, int narrow_blocks, int wide_blocks) {
  LnPlan p{};
  p.vec = can_vec;
  const int step = can_vec ? vec : 1;
  p.wide = d > kLnThreads * narrow;
  const int e = p.wide ? wide : narrow;
  p.tpr = 32;
  while (p.tpr < kLnThreads && p.tpr * e < d) p.tpr *= 2;
  p.cluster = 1;
  if (p.tpr == kLnThreads) {
    while (p.cluster < kLnMaxCluster && p.cluster * kLnThreads * wide < d) p.cluster *= 2;
    while (p.cluster < kLnMaxCluster && rows * p.cluster * 2 <= sms && (int64_t)p.cluster * 2 * kLnThreads * step <= d)
      p.cluster *= 2;
  }
  const int groups = kLnThreads / p.tpr * (p.wide || p.cluster > 1 ? rows_wide : rows_narrow);
  const int64_t need = (rows + groups - 1) / groups;
  const int64_t most = (int64_t)sms * (p.wide || p.cluster > 1 ? wide_blocks : narrow_blocks) / p.cluster;
  p.blocks = (int)(need < most ? need : most);
  if (p.blocks < 1) p.blocks = 1;
  return p;
}

// Sums of N values (1, 2 or 4) over the threads of a row, the same bits in all
// of them. Within a warp the values are halved between the lanes while they
// are added (4 values: 6 shuffles, not 20). `slot` alternates between two
// buffers, so one barrier a reduction suffices: a buffer is written again only
// after the next reduction's barrier.
template <int TPR, bool CL, int N>
struct LnReduce {
  static constexpr int kWarps = kLnThreads / 32;
  struct alignas(16) Smem {
    float warp[2][kWarps][N];
    float cta[2][kLnMaxCluster][N];
  };
  __device__ static __forceinline__ void run(float (&v)[N], Smem* s, int slot) {
    const int lane = threadIdx.x & 31;
    float k = v[0];
    if constexpr (N == 4) {
      const bool up = lane & 16;
      float a = up ? v[2] : v[0], b = up ? v[3] : v[1];
      a += __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16);
      b += __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 16);
      k = (lane & 8 ? b : a) + __shfl_xor_sync(0xffffffffu, lane & 8 ? a : b, 8);
    } else if constexpr (N == 2) {
      k = (lane & 16 ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, lane & 16 ? v[0] : v[1], 16);
    }
    constexpr int kLanes = 32 / N;  // that hold one value between them
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) k += __shfl_xor_sync(0xffffffffu, k, o);
    if constexpr (TPR == 32) {
#pragma unroll
      for (int n = 0; n < N; n++) v[n] = N == 1 ? k : __shfl_sync(0xffffffffu, k, n * kLanes);
    } else {
      const int warp = threadIdx.x >> 5;
      if (lane % kLanes == 0) s->warp[slot][warp][lane / kLanes] = k;
      __syncthreads();
      constexpr int W = TPR / 32;
      const int w0 = warp / W * W;
#pragma unroll
      for (int n = 0; n < N; n++) v[n] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; w++) {
        const Pack<float, N> p = load_pack<float, N>(&s->warp[slot][w0 + w][0]);
#pragma unroll
        for (int n = 0; n < N; n++) v[n] += p.v[n];
      }
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
int ln_launch(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  auto kernel = K::get();
  const int smem = K::smem();
  if (smem > 16384) {  // beside up to 32 KB of static shared memory
    static std::atomic<unsigned> allowed[4];  // a bit per device
    int dev = 0;
    VRS_CUDA(cudaGetDevice(&dev));
    if (dev >= 128 || !(allowed[dev / 32].load() >> (dev % 32) & 1)) {
      VRS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      if (dev < 128) allowed[dev / 32].fetch_or(1u << (dev % 32));
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.blocks * p.cluster + a.col_blocks));
  cfg.blockDim = dim3(kLnThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
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

// The instantiation for a plan.
template <template <class, class, int, int, int, bool> class K, int NARROW, int WIDE, class T, class P, int VEC>
int ln_dispatch_tpr(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  if (p.cluster > 1) return ln_launch<K<T, P, VEC, kLnThreads, WIDE, true>>(a, p, s);
  if (p.wide) return ln_launch<K<T, P, VEC, kLnThreads, WIDE, false>>(a, p, s);
  switch (p.tpr) {
    case 32: return ln_launch<K<T, P, VEC, 32, NARROW, false>>(a, p, s);
    case 64: return ln_launch<K<T, P, VEC, 64, NARROW, false>>(a, p, s);
    case 128: return ln_launch<K<T, P, VEC, 128, NARROW, false>>(a, p, s);
    default: return ln_launch<K<T, P, VEC, 256, NARROW, false>>(a, p, s);
  }
}

template <template <class, class, int, int, int, bool> class K, int NARROW, int WIDE, class T, class P>
int ln_dispatch_vec(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  return p.vec ? ln_dispatch_tpr<K, NARROW, WIDE, T, P, 16 / (int)sizeof(T)>(a, p, s)
               : ln_dispatch_tpr<K, NARROW, WIDE, T, P, 1>(a, p, s);
}

template <template <class, class, int, int, int, bool> class K, int NARROW, int WIDE>
int ln_dispatch(int dtype, int param_dtype, const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  switch (dtype) {
    case VRS_F32: return ln_dispatch_vec<K, NARROW, WIDE, float, float>(a, p, s);
    case VRS_F16:
      return param_dtype == VRS_F32 ? ln_dispatch_vec<K, NARROW, WIDE, f16, float>(a, p, s)
                                    : ln_dispatch_vec<K, NARROW, WIDE, f16, f16>(a, p, s);
    default:
      return param_dtype == VRS_F32 ? ln_dispatch_vec<K, NARROW, WIDE, bf16, float>(a, p, s)
                                    : ln_dispatch_vec<K, NARROW, WIDE, bf16, bf16>(a, p, s);
  }
}

int ln_check(const char* who, int64_t rows, int64_t d, int32_t dtype, int32_t param_dtype);

}  // namespace ops
}  // namespace vrs
