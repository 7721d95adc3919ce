// layer_norm.cuh -- what the layer norm's forward and backward kernels share:
// the launch plan, the split of a row over threads, and its reductions.
//
// A row of d elements is held in registers by TPR threads (4 to 256) of a
// 256-thread block, or by a cluster of 2 to 8 blocks, E elements a thread, so
// that it is read from memory once. Thread tt of a row's TT threads holds the
// vectors i * TT + tt: neighbouring threads read neighbouring 16 bytes.
//
// Rows that 16-byte accesses cannot reach (odd widths, strides or addresses)
// take the same kernels with one element per access. In 16 bits, where a row
// takes a cluster and the rows of every array start alike on or between 4-byte
// words, they take the words that the row lies in: pair i of a thread is columns
// (i * TT + tt) * 2 - shift, shift 1 where rows start between words. With an odd
// stride every other row does, so a block takes rows of one kind only (its
// columns' parameters and sums stay in registers). A word's element beside the
// row counts as zero and is not written; words that reach past the first and the
// last row are read by elements.
#pragma once
#include <cooperative_groups.h>
#include <cuda_pipeline_primitives.h>

#include <atomic>

#include "ops_common.cuh"
#include "tc_common.cuh"

namespace vrs {
namespace ops {

constexpr int kLnThreads = 256;
constexpr int kLnMaxCluster = 8;
constexpr int kLnDevices = 16;  // whose answers are kept
constexpr int64_t kLnMaxD = 32768;
constexpr uint64_t kLnWaitNs = 2000000000ull;
constexpr int kLnWaitCode = 41;

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
  int* err;            // host-visible word that a wait which gave up writes
};

// How a row is held, by its width.
//   small    up to 256 elements: 4 to 32 threads, 8 elements each, two rows at
//            a time (their loads and reductions overlap)
//   narrow   up to 4,096: 32 to 256 threads, 16 elements each
//   between  up to what 128 threads hold, many rows, forward only: 4 to 128
//            threads, 24 elements each, where that leaves fewer idle (45 M elements in bf16: width 136
//            36 us, as small 82; 768 33, as narrow 45; 1,536 35 and 44)
//   wide     up to 8,192, forward only (the backward pass holds five values an
//            element): 256 threads, 32 elements each
//   cluster  the fewest of 2 to 8 blocks (2,248 x 20,016 in bf16: forward 61 us
//            with 3 and backward 136 with 5, powers of two, 4 and 8, 110 and 181), 16
//            elements a thread, or in the forward pass of many rows 32 (fewer
//            blocks to a reduction over a cluster: 3,747 x 12,008 in bf16 57 us
//            with clusters of 2, 80 us with 3)
enum LnClass : int { kLnSmall, kLnNarrow, kLnBetween, kLnWide, kLnCluster, kLnWideCluster };
constexpr int kBetweenBlocks = 2;  // of an SM
constexpr int kSmallE = 8, kSmallRows = 2, kNarrowE = 16, kBetweenE = 24, kWideE = 32;

enum LnAccess : int { kLnElements, kLn16Bytes, kLnPairs };

struct LnPlan {
  LnClass cls;
  int tpr;      // threads of a row within a block (4..256)
  int cluster;  // blocks of a row (1: none)
  LnAccess access;
  int blocks;   // grid, in clusters: at most so many
};

// The fewest threads that hold a row; a row wider than one block takes a
// cluster, and so do rows so few that blocks alone would leave SMs idle (each
// thread still has at least one access).
// Pairs pay where a row takes a cluster (5,492 x 8,193 in bf16: backward 265 us
// and by elements 393; 43,988 x 1,023 the other way 96 and 81).
inline LnPlan ln_plan(int64_t rows, int d, bool allow_wide, int vec, LnAccess access, int sms, int blocks_per_sm) {
  const int d_given = d;
  LnPlan p{};
  p.access = access;
  const int step = access == kLn16Bytes ? vec : access == kLnPairs ? 2 : 1;
  if (access == kLnPairs) d++;  // columns from -1
  p.cluster = 1;
  if (d <= 32 * kSmallE) {
    p.cls = kLnSmall;
    p.tpr = 4;
    while (p.tpr * kSmallE < d) p.tpr *= 2;
  } else if (d <= kLnThreads * kNarrowE) {
    p.cls = kLnNarrow;
    p.tpr = 32;
    while (p.tpr * kNarrowE < d) p.tpr *= 2;
  } else {
    p.cls = kLnCluster;
    p.tpr = kLnThreads;
    p.cluster = (d + kLnThreads * kNarrowE - 1) / (kLnThreads * kNarrowE);
    if (allow_wide && rows * p.cluster > sms) {
      p.cluster = (d + kLnThreads * kWideE - 1) / (kLnThreads * kWideE);
      p.cls = p.cluster > 1 ? kLnWideCluster : kLnWide;
    }
  }
  if (allow_wide && d <= kLnThreads / 2 * kBetweenE) {
    int t = 4;
    while (t * kBetweenE < d) t *= 2;
    if (t * kBetweenE < p.tpr * (p.cls == kLnSmall ? kSmallE : kNarrowE) && rows * t > (int64_t)sms * kLnThreads) {
      p.cls = kLnBetween;
      p.tpr = t;
      blocks_per_sm = kBetweenBlocks;
    }
  }
  if (p.tpr == kLnThreads && rows * p.cluster <= sms) {
    while (p.cluster * 2 <= kLnMaxCluster && rows * p.cluster <= sms &&
           (int64_t)p.cluster * 2 * kLnThreads * step <= d)
      p.cluster *= 2;
    if (p.cluster > 1) p.cls = kLnCluster;
  }
  if (access == kLnPairs && p.cluster == 1)
    return ln_plan(rows, d_given, allow_wide, vec, kLnElements, sms, blocks_per_sm);
  const int at_once = kLnThreads / p.tpr * (p.cls == kLnSmall ? kSmallRows : 1);
  const int64_t need = (rows + at_once - 1) / at_once;
  const int64_t most = (int64_t)sms * blocks_per_sm / p.cluster;
  p.blocks = (int)(need < most ? need : most);
  if (access == kLnPairs) p.blocks = (p.blocks + 1) / 2 * 2;  // a half for each kind of rows
  if (p.blocks < 1) p.blocks = 1;
  return p;
}

// How the rows of N arrays of T's size can be reached.
struct LnRows {
  const void* p;
  int64_t stride;
};
template <int N>
LnAccess ln_access(const LnRows (&in)[N], int64_t rows, int64_t d, int bytes, bool params16) {
  const int vec = 16 / bytes;
  bool whole = d % vec == 0 && params16, alike = bytes == 2 && d < kLnMaxD;  // (column -1 takes a place)
  for (const LnRows& r : in) {
    whole = whole && aligned16(r.p) && (rows == 1 || r.stride % vec == 0);
    alike = alike && (((uintptr_t)r.p ^ (uintptr_t)in[0].p) & 2) == 0 && (rows == 1 || (r.stride - in[0].stride) % 2 == 0);
  }
  return whole ? kLn16Bytes : alike ? kLnPairs : kLnElements;
}

// Which of its columns a thread holds, and which rows its block takes.
template <int VEC>
struct LnPlace {
  static constexpr bool kPairs = VEC == 2;
  int tt, TT, shift, d;
  int64_t first;  // the block's first row
  __device__ __forceinline__ int column(int i) const { return (i * TT + tt) * VEC - (kPairs ? shift : 0); }
  // Whether element j of access i is one of the row's.
  __device__ __forceinline__ bool has(int i, int j) const {
    const int c = column(i) + j;
    return c < d && (!kPairs || c >= 0);
  }
  // Block `block` of `groups` rows a turn, thread group g: the first row.
  __device__ __forceinline__ int64_t start(const LnArgs& a, int64_t block, int groups, int g) {
    d = a.d;
    shift = 0;
    if constexpr (kPairs) {
      shift = (int)(((uintptr_t)a.x >> 1) + (uintptr_t)((block & 1) * a.xs)) & 1;
      first = (block >> 1) * 2 * groups + (block & 1);
      return first + 2 * g;
    }
    first = block * groups;
    return first + g;
  }
  // The parameters of the thread's columns.
  template <class P, int E>
  __device__ __forceinline__ void load(Held<P, E, VEC>& h, const void* p) const {
    if (!p) return;
#pragma unroll
    for (int i = 0; i < E / VEC; i++) {
      if constexpr (kPairs) {
#pragma unroll
        for (int j = 0; j < 2; j++)
          if (has(i, j)) h.k[i].v[j] = ((const P*)p)[column(i) + j];
      } else {
        if (column(i) < d) h.load(i, (const P*)p + column(i));
      }
    }
  }
  template <class T, int E>
  __device__ __forceinline__ void store(T* row, const F2 (&v)[E / 2]) const {
#pragma unroll
    for (int i = 0; i < E / VEC; i++) {
      const int c = column(i);
      if constexpr (kPairs) {
        if (c >= 0 && c + 1 < d) {
          store_held<T, VEC, E>(row + c, v, i);
        } else if (c < d) {
          float lo, hi;
          unpack_f2(v[i], lo, hi);
          if (c >= 0) row[c] = from_f32<T>(lo);
          if (c + 1 < d) row[c + 1] = from_f32<T>(hi);
        }
      } else {
        if (c < d) store_held<T, VEC, E>(row + c, v, i);
      }
    }
  }
};

// Sums of N values (1, 2 or 4) over the threads of a row, the same bits in all
// of them. Within a warp the values are halved between the lanes while they
// are added (4 values: 6 shuffles, not 20). `slot` alternates between two
// buffers, so one barrier a reduction suffices: a buffer is written again only
// after the next reduction's barrier.
//
// Between the blocks of a cluster the sums travel as asynchronous stores that
// complete on a barrier of the block they go to. (A cluster barrier in their
// place would wait for each thread's own stores of the row before: 2,746 x
// 16,384 in bf16 forward 61 and 46 us, backward 146 and 124.)
// A block sends its next-but-one sums only after it has all blocks' next ones,
// which they send after they have read the last ones: two buffers suffice here
// too. A wait that gives up says so and goes on with NaN, so that all threads
// take the same turns.
template <int TPR, bool CL, int N>
struct LnReduce {
  static constexpr int kWarps = kLnThreads / 32;
  struct alignas(16) Smem {
    float warp[2][kWarps][N];
    float cta[2][kLnMaxCluster][N];
    alignas(8) uint64_t bar[2];
    volatile int abort;
  };
  // Before the first reduction, by all threads of a cluster.
  __device__ static __forceinline__ void start(Smem* s) {
    if constexpr (CL) {
      if (threadIdx.x == 0) {
        tc::mbar_init(&s->bar[0], 1);
        tc::mbar_init(&s->bar[1], 1);
        s->abort = 0;
        tc::fence_mbar_init();
      }
      cooperative_groups::this_cluster().sync();
    }
  }
  // The turn-th reduction.
  __device__ static __forceinline__ void run(float (&v)[N], Smem* s, int turn, int* err) {
    const int slot = turn & 1;
    if constexpr (TPR < 32) {
#pragma unroll
      for (int o = TPR / 2; o > 0; o >>= 1)
#pragma unroll
        for (int n = 0; n < N; n++) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
      return;
    }
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
      static_assert(N <= 2, "sums of one row");
      auto cluster = cooperative_groups::this_cluster();
      const int c = (int)cluster.num_blocks(), r = (int)cluster.block_rank();
      if ((int)threadIdx.x < c && !s->abort) {
        if (threadIdx.x == 0) tc::mbar_expect_tx(&s->bar[slot], c * N * 4);
        const uint32_t to = tc::mapa_shared(&s->cta[slot][r][0], threadIdx.x);
        const uint32_t bar = tc::mapa_shared(&s->bar[slot], threadIdx.x);
        if constexpr (N == 1)
          asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(to), "f"(v[0]),
                       "r"(bar)
                       : "memory");
        else
          asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to),
                       "f"(v[0]), "f"(v[N - 1]), "r"(bar)
                       : "memory");
      }
      const bool ok = tc::mbar_try_wait(&s->bar[slot], turn >> 1 & 1) ||
                      (!s->abort && tc::mbar_wait(&s->bar[slot], turn >> 1 & 1, &s->abort, err, kLnWaitCode, kLnWaitNs));
#pragma unroll
      for (int n = 0; n < N; n++) v[n] = ok ? 0.0f : NAN;
      for (int b = 0; b < c; b++)
#pragma unroll
        for (int n = 0; n < N; n++) v[n] += s->cta[slot][b][n];
    }
  }
};

// A ring in shared memory for the rows a thread will hold next: asynchronous
// copies of 16 bytes, a pair or a 32-bit element into slots of its own (nobody
// else reads them, so no barrier is added), DEPTH - 1 turns ahead. R rows and
// ARRAYS arrays a turn. Columns past the row's end are zeros and stay so. Single
// 32-bit elements are copied so where a row takes a cluster, whose turns are long
// (5,492 x 8,193 forward in f32 162 us; in bf16 by elements, which are loaded
// when needed, 227), and loaded when needed elsewhere (43,988 x 1,023 backward in
// f32 98 us, copied 117).
template <class T, int VEC, int E, int R, int ARRAYS, bool CL>
struct LnRing {
  static constexpr int NV = E / VEC;
  static constexpr int kUnit = VEC * (int)sizeof(T);  // bytes of a copy
  static constexpr bool kAsync = VEC > 1 || (CL && kUnit >= 4);
  using Unit = Pack<uint32_t, kAsync ? kUnit / 4 : 1>;
  static constexpr int kStage = R * ARRAYS * E * (int)sizeof(T) * kLnThreads;  // bytes of a turn
  static constexpr int kDepth = kStage <= 16384 ? 3 : 2;
  static constexpr int kBytes = kAsync ? kDepth * kStage : 0;

  const T* base[ARRAYS];
  int64_t stride[ARRAYS];
  int64_t rows;
  int64_t apart;  // rows between those of a turn; a turn is R times as long
  LnPlace<VEC> at_columns;
  int at;

  __device__ __forceinline__ Unit* slot(int k, int r, int array, int i) const {
    extern __shared__ uint4 s_ring[];
    return reinterpret_cast<Unit*>(s_ring) + (((k * R + r) * ARRAYS + array) * NV + i) * kLnThreads + threadIdx.x;
  }
  // A pair one of whose elements lies before the first row or after the last:
  // its other element.
  __device__ __forceinline__ bool outside(int c, int64_t row) const {
    return (c < 0 && row == 0) || (c + 1 == at_columns.d && row + 1 == rows);
  }
  __device__ __forceinline__ Pack<T, VEC> inner(const T* p, int c) const {
    Pack<T, VEC> q = {};
    if (c >= 0) q.v[0] = p[c];
    if (c + 1 < at_columns.d) q.v[VEC - 1] = p[c + 1];
    return q;
  }
  __device__ __forceinline__ void fetch(int64_t row, int k) const {
    if constexpr (kAsync) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        if (row + r * apart < rows) {
#pragma unroll
          for (int m = 0; m < ARRAYS; m++) {
            const int64_t at_row = row + r * apart;
            const T* p = base[m] + at_row * stride[m];
#pragma unroll
            for (int i = 0; i < NV; i++) {
              const int c = at_columns.column(i);
              if (c >= at_columns.d) continue;
              if constexpr (VEC == 2) {
                if (outside(c, at_row)) {
                  *reinterpret_cast<Pack<T, 2>*>(slot(k, r, m, i)) = inner(p, c);
                  continue;
                }
              }
              __pipeline_memcpy_async(slot(k, r, m, i), p + c, kUnit);
            }
          }
        }
      }
      __pipeline_commit();
    }
  }
  __device__ __forceinline__ void start(int64_t row) {
    at = 0;
    if constexpr (kAsync) {
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (at_columns.column(i) >= at_columns.d)
          for (int k = 0; k < kDepth * R * ARRAYS; k++)
            *slot(k / (R * ARRAYS), k / ARRAYS % R, k % ARRAYS, i) = Unit{};
      for (int k = 0; k < kDepth - 1; k++) fetch(row + k * R * apart, k);
    }
  }
  // Starts the copies of a later turn and waits for those of `row`'s.
  __device__ __forceinline__ void next(int64_t row) {
    if constexpr (kAsync) {
      fetch(row + (kDepth - 1) * R * apart, at == 0 ? kDepth - 1 : at - 1);
      __pipeline_wait_prior(kDepth - 1);
    }
  }
  __device__ __forceinline__ void done() { at = at + 1 == kDepth ? 0 : at + 1; }
  // Row r of the turn at `row`; zeros past the last row.
  __device__ __forceinline__ Held<T, E, VEC> get(int64_t row, int r, int m) const {
    Held<T, E, VEC> h;
    h.fill(0.0f);
    if (row + r * apart < rows) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int c = at_columns.column(i);
        if constexpr (kAsync)
          h.k[i] = *reinterpret_cast<const Pack<T, VEC>*>(slot(at, r, m, i));
        else if (c < at_columns.d)
          h.load(i, base[m] + (row + r * apart) * stride[m] + c);
        if constexpr (VEC == 2) {  // the element before or after the row
          uint32_t& u = *reinterpret_cast<uint32_t*>(&h.k[i]);
          if (i == 0 && c < 0) u &= 0xffff0000u;
          if (c + 1 == at_columns.d) u &= 0xffffu;
        }
      }
    }
    return h;
  }
  __device__ __forceinline__ void drain() const {
    if constexpr (kAsync) __pipeline_wait_prior(0);
  }
};

// Clusters take the rows in turn, so no more are launched than run at a time (an
// SM group of the device holds whole clusters only: 1,373 x 32,767 in bf16,
// backward 203 us, with as many as the SMs' sum would hold 316); p.blocks says
// how many.
template <class K>
int ln_launch(const LnArgs& a, LnPlan& p, cudaStream_t s) {
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
  cfg.blockDim = dim3(kLnThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (p.cluster > 1) {
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)p.cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
    static std::atomic<int> active[kLnDevices][kLnMaxCluster + 1];  // zero: not asked yet
    int dev = 0;
    VRS_CUDA(cudaGetDevice(&dev));
    int n = dev < kLnDevices ? active[dev][p.cluster].load() : 0;
    if (n == 0) {
      cfg.gridDim = dim3((unsigned)p.cluster);
      VRS_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
      if (n < 1) n = 1;
      if (dev < kLnDevices) active[dev][p.cluster].store(n);
    }
    if (p.access == kLnPairs) n = n < 2 ? 2 : n / 2 * 2;
    if (p.blocks > n) p.blocks = n;
  }
  cfg.gridDim = dim3((unsigned)(p.blocks * p.cluster + a.col_blocks));
  VRS_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  count_launch();
  return VRS_OK;
}

// The instantiation for a plan: K<T, P, VEC, TPR, E, R, CL>.
template <template <class, class, int, int, int, int, bool> class K, bool WIDE, class T, class P, int VEC>
int ln_dispatch_tpr(const LnArgs& a, LnPlan& p, cudaStream_t s) {
  if (p.cls == kLnCluster) return ln_launch<K<T, P, VEC, kLnThreads, kNarrowE, 1, true>>(a, p, s);
  if constexpr (WIDE) {
    if (p.cls == kLnWideCluster) return ln_launch<K<T, P, VEC, kLnThreads, kWideE, 1, true>>(a, p, s);
    if (p.cls == kLnWide) return ln_launch<K<T, P, VEC, kLnThreads, kWideE, 1, false>>(a, p, s);
  }
  if constexpr (WIDE)
    if (p.cls == kLnBetween) switch (p.tpr) {
        case 4: return ln_launch<K<T, P, VEC, 4, kBetweenE, 1, false>>(a, p, s);
        case 8: return ln_launch<K<T, P, VEC, 8, kBetweenE, 1, false>>(a, p, s);
        case 16: return ln_launch<K<T, P, VEC, 16, kBetweenE, 1, false>>(a, p, s);
        case 32: return ln_launch<K<T, P, VEC, 32, kBetweenE, 1, false>>(a, p, s);
        case 64: return ln_launch<K<T, P, VEC, 64, kBetweenE, 1, false>>(a, p, s);
        default: return ln_launch<K<T, P, VEC, 128, kBetweenE, 1, false>>(a, p, s);
      }
  if (p.cls == kLnSmall) switch (p.tpr) {
      case 4: return ln_launch<K<T, P, VEC, 4, kSmallE, kSmallRows, false>>(a, p, s);
      case 8: return ln_launch<K<T, P, VEC, 8, kSmallE, kSmallRows, false>>(a, p, s);
      case 16: return ln_launch<K<T, P, VEC, 16, kSmallE, kSmallRows, false>>(a, p, s);
      default: return ln_launch<K<T, P, VEC, 32, kSmallE, kSmallRows, false>>(a, p, s);
    }
  switch (p.tpr) {
    case 32: return ln_launch<K<T, P, VEC, 32, kNarrowE, 1, false>>(a, p, s);
    case 64: return ln_launch<K<T, P, VEC, 64, kNarrowE, 1, false>>(a, p, s);
    case 128: return ln_launch<K<T, P, VEC, 128, kNarrowE, 1, false>>(a, p, s);
    default: return ln_launch<K<T, P, VEC, 256, kNarrowE, 1, false>>(a, p, s);
  }
}

template <template <class, class, int, int, int, int, bool> class K, bool WIDE, class T, class P>
int ln_dispatch_vec(const LnArgs& a, LnPlan& p, cudaStream_t s) {
  if (p.access == kLn16Bytes) return ln_dispatch_tpr<K, WIDE, T, P, 16 / (int)sizeof(T)>(a, p, s);
  if constexpr (sizeof(T) == 2) {
    if (p.access == kLnPairs) {
      if constexpr (WIDE)
        if (p.cls == kLnWideCluster) return ln_launch<K<T, P, 2, kLnThreads, kWideE, 1, true>>(a, p, s);
      return ln_launch<K<T, P, 2, kLnThreads, kNarrowE, 1, true>>(a, p, s);
    }
  }
  return ln_dispatch_tpr<K, WIDE, T, P, 1>(a, p, s);
}

template <template <class, class, int, int, int, int, bool> class K, bool WIDE>
int ln_dispatch(int dtype, int param_dtype, const LnArgs& a, LnPlan& p, cudaStream_t s) {
  switch (dtype) {
    case VRS_F32: return ln_dispatch_vec<K, WIDE, float, float>(a, p, s);
    case VRS_F16:
      return param_dtype == VRS_F32 ? ln_dispatch_vec<K, WIDE, f16, float>(a, p, s)
                                    : ln_dispatch_vec<K, WIDE, f16, f16>(a, p, s);
    default:
      return param_dtype == VRS_F32 ? ln_dispatch_vec<K, WIDE, bf16, float>(a, p, s)
                                    : ln_dispatch_vec<K, WIDE, bf16, bf16>(a, p, s);
  }
}

int ln_check(const char* who, int64_t rows, int64_t d, int32_t dtype, int32_t param_dtype);

}  // namespace ops
}  // namespace vrs
