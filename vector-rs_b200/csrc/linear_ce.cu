// linear_ce.cu -- softmax cross entropy of scale * x table^T against one
// target a row, without keeping the scores, and its gradients:
//   z = scale x w_v, lse = log sum_v e^z, loss = lse - z[target]
//   g = (e^(z - lse) - [v = target]) dloss scale, dx = g table, dtable = g^T x.
// A row whose target lies outside the table takes no part: loss 0, lse 0, no
// gradient, whatever its values are.
//
// CUDA-core tiles (64 x 64, 16 deep), the classes taken in pieces whose
// gradient of the scores fits a fixed workspace.
#include <cmath>

#include "ops_common.cuh"

namespace vrs {
namespace ops {
namespace {

constexpr int BT = 64, BK = 16;
constexpr int64_t kPieceBytes = 256ll << 20;

struct CeArgs {
  const void* x;
  const void* w;
  int64_t xs, ws;
  int64_t rows, classes;
  int d;
  const int64_t* targets;
  float scale;
  float2* part;  // [row][tile]: maximum and sum of e^(z - maximum)
  int64_t ntiles;
  float* zt;
  const float* lse;
  const float* dloss;
  float* g;  // [rows][piece]
  int64_t v0, vn, gp;
};

__device__ __forceinline__ bool takes_part(const CeArgs& a, int64_t r) {
  return r < a.rows && a.targets[r] >= 0 && a.targets[r] < a.classes;
}

// One 64 x 64 tile of the scores; 256 threads, 4 x 4 each. GRAD: the gradient
// of the scores, else each row's maximum and sum over the tile.
template <class T, bool GRAD>
__global__ void __launch_bounds__(256) ce_tile_kernel(const CeArgs a) {
  __shared__ float sx[BK][BT + 1], sw[BK][BT + 1];
  __shared__ float sz[BT][BT + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t m0 = (int64_t)blockIdx.y * BT, n0 = a.v0 + (int64_t)blockIdx.x * BT, n1 = a.v0 + a.vn;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.d; k0 += BK) {
    for (int i = threadIdx.x; i < BT * BK; i += 256) {
      const int k = i % BK, r = i / BK;
      const int64_t m = m0 + r, n = n0 + r;
      sx[k][r] = m < a.rows && k0 + k < a.d ? to_f32(((const T*)a.x)[m * a.xs + k0 + k]) : 0.0f;
      sw[k][r] = n < n1 && k0 + k < a.d ? to_f32(((const T*)a.w)[n * a.ws + k0 + k]) : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < BK; k++)
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sx[k][ty * 4 + i], sw[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      const float z = acc[i][j] * a.scale;
      if (GRAD) {
        if (m >= a.rows || n >= n1) continue;
        float g = 0.0f;
        if (takes_part(a, m)) g = (expf(z - a.lse[m]) - (a.targets[m] == n ? 1.0f : 0.0f)) * a.dloss[m] * a.scale;
        a.g[m * a.gp + n - a.v0] = g;
      } else {
        sz[ty * 4 + i][tx * 4 + j] = n < n1 ? z : -INFINITY;
        if (m < a.rows && n < n1 && a.targets[m] == n) a.zt[m] = z;
      }
    }
  if (GRAD) return;
  __syncthreads();
  const int64_t m = m0 + threadIdx.x;
  if (threadIdx.x < BT && m < a.rows) {
    float top = -INFINITY, sum = 0.0f;
    for (int j = 0; j < BT; j++) top = fmaxf(top, sz[threadIdx.x][j]);
    const float sub = top == -INFINITY ? 0.0f : top;
    for (int j = 0; j < BT; j++) sum += expf(sz[threadIdx.x][j] - sub);
    a.part[m * a.ntiles + blockIdx.x] = make_float2(top, sum);
  }
}

// loss and lse from the tiles' maxima and sums: one warp a row.
__global__ void ce_combine_kernel(const CeArgs a, float* loss, float* lse) {
  const int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (r >= a.rows) return;
  const bool in = takes_part(a, r);
  float top = -INFINITY, sum = 0.0f;
  if (in) {
    for (int64_t t = lane; t < a.ntiles; t += 32) top = fmaxf(top, a.part[r * a.ntiles + t].x);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float sub = top == -INFINITY ? 0.0f : top;
    for (int64_t t = lane; t < a.ntiles; t += 32) {
      const float2 p = a.part[r * a.ntiles + t];
      sum += p.y * expf((p.x == -INFINITY ? 0.0f : p.x) - sub);
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  }
  if (lane == 0) {
    const float l = in ? top + logf(sum) : 0.0f;
    lse[r] = l;
    loss[r] = in ? l - a.zt[r] : 0.0f;
  }
}

// acc[m][n] (+)= sum_k a[m am + k ak] b[n bn + k bk]; rows of b whose target
// lies outside the table (`skip`, along k) are left out.
template <class T>
__global__ void __launch_bounds__(256)
    ce_product_kernel(const float* a, int64_t am, int64_t ak, const T* b, int64_t bn, int64_t bk, int64_t M, int64_t N,
                      int64_t K, CeArgs c, bool skip, float* acc, bool add, T* out, int64_t os) {
  __shared__ float sa[BK][BT + 1], sb[BK][BT + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t m0 = (int64_t)blockIdx.y * BT, n0 = (int64_t)blockIdx.x * BT;
  float s[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += BK) {
    for (int i = threadIdx.x; i < BT * BK; i += 256) {
      const int r = i % BT, k = i / BT;
      const int64_t m = m0 + r, n = n0 + r, kk = k0 + k;
      const bool in = kk < K && (!skip || takes_part(c, kk));
      sa[k][r] = in && m < M ? a[m * am + kk * ak] : 0.0f;
      sb[k][r] = in && n < N ? to_f32(b[n * bn + kk * bk]) : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < BK; k++)
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) s[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], s[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= M || n >= N) continue;
      if (acc) acc[m * N + n] = (add ? acc[m * N + n] : 0.0f) + s[i][j];
      else out[m * os + n] = from_f32<T>(s[i][j]);
    }
}

// dx from its 32-bit sums; rows that take no part get zeros.
template <class T>
__global__ void ce_finish_kernel(const CeArgs a, const float* acc, T* out, int64_t os) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.rows * a.d) return;
  const int64_t r = i / a.d, c = i % a.d;
  out[r * os + c] = takes_part(a, r) ? from_f32<T>(acc[i]) : from_f32<T>(0.0f);
}

int64_t piece_of(int64_t rows, int64_t classes) {
  int64_t vc = kPieceBytes / (4 * rows) / BT * BT;
  vc = vc < BT ? BT : vc;
  return vc < classes ? vc : classes;
}

int64_t up(int64_t b) { return (b + 255) / 256 * 256; }

int check(const char* who, int64_t rows, int64_t classes, int64_t d, int32_t dtype) {
  if (dtype != VRS_F16 && dtype != VRS_BF16)
    return invalid(std::string(who) + ": rows and table are f16 or bf16 (operands of the tensor cores)");
  if (rows < 0 || rows > (1ll << 31) - 512) return invalid(std::string(who) + ": rows must be in 0..2^31-512");
  if (classes < 1 || classes > (1ll << 31) - 512) return invalid(std::string(who) + ": classes must be in 1..2^31-512");
  if (d < 1 || d > 65536) return invalid(std::string(who) + ": d must be in 1..65536");
  return VRS_OK;
}

template <class T>
int backward(CeArgs a, void* dx, int64_t dxs, void* dtable, int64_t dts, char* ws, cudaStream_t s) {
  const int64_t piece = piece_of(a.rows, a.classes);
  a.g = (float*)ws;
  a.gp = piece;
  float* acc = (float*)(ws + up(a.rows * piece * 4));
  for (a.v0 = 0; a.v0 < a.classes; a.v0 += piece) {
    a.vn = a.classes - a.v0 < piece ? a.classes - a.v0 : piece;
    const unsigned tv = (unsigned)((a.vn + BT - 1) / BT), tr = (unsigned)((a.rows + BT - 1) / BT),
                   td = (unsigned)((a.d + BT - 1) / BT);
    ce_tile_kernel<T, true><<<dim3(tv, tr), 256, 0, s>>>(a);
    if (dx)
      ce_product_kernel<T><<<dim3(td, tr), 256, 0, s>>>(a.g, a.gp, 1, (const T*)a.w + a.v0 * a.ws, 1, a.ws, a.rows,
                                                        a.d, a.vn, a, false, acc, a.v0 > 0, nullptr, 0);
    if (dtable)
      ce_product_kernel<T><<<dim3(td, tv), 256, 0, s>>>(a.g, 1, a.gp, (const T*)a.x, 1, a.xs, a.vn, a.d, a.rows, a,
                                                        true, nullptr, false, (T*)dtable + a.v0 * dts, dts);
    count_launch(3);
  }
  if (dx) {
    ce_finish_kernel<T><<<(unsigned)((a.rows * a.d + 255) / 256), 256, 0, s>>>(a, acc, (T*)dx, dxs);
    count_launch();
  }
  VRS_CUDA(cudaGetLastError());
  return VRS_OK;
}

int64_t need_bytes(int64_t rows, int64_t classes, int64_t d, bool back) {
  if (rows == 0) return 0;
  const int64_t fwd = up(rows * ((classes + BT - 1) / BT) * 8) + up(rows * 4);
  return back ? up(rows * piece_of(rows, classes) * 4) + up(rows * d * 4) : fwd;
}

}  // namespace
}  // namespace ops
}  // namespace vrs

extern "C" int vrs_linear_cross_entropy_workspace(int64_t rows, int64_t classes, int64_t d, int32_t dtype,
                                                  int32_t backward, int32_t aligned, int64_t* out_bytes) {
  using namespace vrs::ops;
  (void)aligned;
  if (!out_bytes) return invalid("vrs_linear_cross_entropy_workspace: null out_bytes");
  VRS_TRY(check("vrs_linear_cross_entropy_workspace", rows, classes, d, dtype));
  *out_bytes = need_bytes(rows, classes, d, backward != 0);
  return VRS_OK;
}

extern "C" int vrs_linear_cross_entropy_forward(const void* x, int64_t x_stride, int64_t rows, const void* table,
                                                int64_t table_stride, int64_t classes, int64_t d, int32_t dtype,
                                                const int64_t* targets, float scale, float* loss, float* lse,
                                                void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  const char* who = "vrs_linear_cross_entropy_forward";
  VRS_TRY(check(who, rows, classes, d, dtype));
  if (!(scale > 0.0f) || !std::isfinite(scale)) return invalid(std::string(who) + ": scale must be positive and finite");
  if (rows == 0) return VRS_OK;
  if (!x || !table || !targets || !loss || !lse || !workspace) return invalid(std::string(who) + ": null buffer");
  if ((rows > 1 && x_stride < d) || (classes > 1 && table_stride < d))
    return invalid(std::string(who) + ": row strides must be at least d");
  if ((uintptr_t)workspace % 256) return invalid(std::string(who) + ": workspace must be 256-byte aligned");
  if (workspace_bytes < need_bytes(rows, classes, d, false)) return invalid(std::string(who) + ": workspace too small");
  CeArgs a{};
  a.x = x; a.w = table; a.xs = x_stride; a.ws = table_stride;
  a.rows = rows; a.classes = classes; a.d = (int)d; a.targets = targets; a.scale = scale;
  a.ntiles = (classes + BT - 1) / BT;
  a.part = (float2*)workspace;
  a.zt = (float*)((char*)workspace + up(rows * a.ntiles * 8));
  a.v0 = 0; a.vn = classes;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  const dim3 grid((unsigned)a.ntiles, (unsigned)((rows + BT - 1) / BT));
  if (dtype == VRS_F16) ce_tile_kernel<f16, false><<<grid, 256, 0, s>>>(a);
  else ce_tile_kernel<bf16, false><<<grid, 256, 0, s>>>(a);
  ce_combine_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(a, loss, lse);
  count_launch(2);
  VRS_CUDA(cudaGetLastError());
  return VRS_OK;
}

extern "C" int vrs_linear_cross_entropy_backward(const float* dloss, const void* x, int64_t x_stride, int64_t rows,
                                                 const void* table, int64_t table_stride, int64_t classes, int64_t d,
                                                 int32_t dtype, const int64_t* targets, float scale, const float* lse,
                                                 void* dx, int64_t dx_stride, void* dtable, int64_t dtable_stride,
                                                 void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  const char* who = "vrs_linear_cross_entropy_backward";
  VRS_TRY(check(who, rows, classes, d, dtype));
  if (!(scale > 0.0f) || !std::isfinite(scale)) return invalid(std::string(who) + ": scale must be positive and finite");
  if ((rows > 1 && (x_stride < d || (dx && dx_stride < d))) ||
      (classes > 1 && (table_stride < d || (dtable && dtable_stride < d))))
    return invalid(std::string(who) + ": row strides must be at least d");
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (rows == 0) {
    if (dtable) VRS_CUDA(cudaMemset2DAsync(dtable, (classes > 1 ? dtable_stride : d) * 2, 0, d * 2, classes, s));
    return VRS_OK;
  }
  if (!dx && !dtable) return VRS_OK;
  if (!dloss || !x || !table || !targets || !lse || !workspace) return invalid(std::string(who) + ": null buffer");
  if ((uintptr_t)workspace % 256) return invalid(std::string(who) + ": workspace must be 256-byte aligned");
  if (workspace_bytes < need_bytes(rows, classes, d, true)) return invalid(std::string(who) + ": workspace too small");
  CeArgs a{};
  a.x = x; a.w = table; a.xs = x_stride; a.ws = table_stride;
  a.rows = rows; a.classes = classes; a.d = (int)d; a.targets = targets; a.scale = scale;
  a.lse = lse; a.dloss = dloss;
  return dtype == VRS_F16 ? backward<f16>(a, dx, dx_stride, dtable, dtable_stride, (char*)workspace, s)
                          : backward<bf16>(a, dx, dx_stride, dtable, dtable_stride, (char*)workspace, s);
}
