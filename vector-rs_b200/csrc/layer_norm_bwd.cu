// layer_norm_bwd.cu -- gradients of the layer norm. With xh = (x - mean) rstd
// and g = dy * weight, per row
//   dx = rstd (g - mean(g) - xh mean(g xh)),
// and over all rows dweight = sum dy xh, dbias = sum dy.
//
// Bound by memory: x and dy in, dx out, 3 d elements a row. One kernel reads
// them once: a row's two means need one joint reduction, and each thread keeps
// the parameter sums of its own columns in 32-bit registers over all the rows
// its block takes. The blocks' sums go to a [blocks][2][d] array that a second
// kernel adds in block order, so the result does not depend on timing.
#include "layer_norm.cuh"

namespace vrs {
namespace ops {
namespace {

// Elements a thread holds: x and dy of a row and two column sums each.
constexpr int kE = 16;
constexpr int kBlocksPerSm = 2;

template <class T, class P, int VEC, int TPR, bool CL>
__global__ void __launch_bounds__(kLnThreads, kBlocksPerSm) ln_bwd_kernel(const LnArgs a) {
  constexpr int NV = kE / VEC, GROUPS = kLnThreads / TPR;
  using Red = LnReduce<TPR, CL, 2>;
  __shared__ typename Red::Smem s_red;
  __shared__ float s_col[GROUPS > 1 ? 2 * TPR * kE : 1];
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
  const T* dy = (const T*)a.dy;
  T* dx = (T*)a.y;
  const P* w = (const P*)a.weight;
  const float inv_d = 1.0f / (float)a.d;
  float dw[kE], db[kE];
#pragma unroll
  for (int e = 0; e < kE; e++) dw[e] = db[e] = 0.0f;
  int slot = 0;
  for (int64_t r0 = first * GROUPS; r0 < a.rows; r0 += step * GROUPS) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool have = row < a.rows;
    Pack<T, VEC> kx[NV], ky[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (i * TT + tt) * VEC;
      if (have && c < a.d) {
        kx[i] = load_pack<T, VEC>(x + row * a.xs + c);
        ky[i] = load_pack<T, VEC>(dy + row * a.dys + c);
      }
    }
    const float mean = have ? a.mean_in[row] : 0.0f, rstd = have ? a.rstd_in[row] : 0.0f;
    float xh[kE], g[kE];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (i * TT + tt) * VEC;
      if (have && c < a.d) {
        float f[VEC];
        if (w) load_params<P, VEC>(w + c, f);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const int e = i * VEC + j;
          const float d_y = to_f32(ky[i].v[j]);
          xh[e] = (to_f32(kx[i].v[j]) - mean) * rstd;
          dw[e] = fmaf(d_y, xh[e], dw[e]);
          db[e] += d_y;
          g[e] = w ? d_y * f[j] : d_y;
          s[0] += g[e];
          s[1] = fmaf(g[e], xh[e], s[1]);
        }
      }
    }
    Red::run(s, &s_red, slot);
    slot ^= 1;
    const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (i * TT + tt) * VEC;
      if (have && c < a.d) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) o[j] = rstd * (g[i * VEC + j] - fmaf(xh[i * VEC + j], m1, m0));
        store_pack<T, VEC>(dx + row * a.ys + c, o);
      }
    }
  }
  if (a.partial) {
    float* out = a.partial + first * 2 * a.d;
    if constexpr (GROUPS > 1) {
      // The groups of a block add their sums in turn (always in this order).
      for (int g = 0; g < GROUPS; g++) {
        if ((int)threadIdx.x / TPR == g) {
#pragma unroll
          for (int i = 0; i < NV; i++) {
            const int c = (i * TT + tt) * VEC;
            if (c < a.d) {
#pragma unroll
              for (int j = 0; j < VEC; j++) {
                float* q = s_col + c + j;
                q[0] = (g ? q[0] : 0.0f) + dw[i * VEC + j];
                q[TPR * kE] = (g ? q[TPR * kE] : 0.0f) + db[i * VEC + j];
              }
            }
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < a.d; c += kLnThreads) {
        out[c] = s_col[c];
        out[a.d + c] = s_col[TPR * kE + c];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int c = (i * TT + tt) * VEC;
        if (c < a.d) {
#pragma unroll
          for (int j = 0; j < VEC; j++) {
            out[c + j] = dw[i * VEC + j];
            out[a.d + c + j] = db[i * VEC + j];
          }
        }
      }
    }
  }
  // A block must not leave while another still writes its shared memory.
  if constexpr (CL) cooperative_groups::this_cluster().sync();
}

template <class T, class P, int VEC, int TPR, bool CL>
struct BwdKernel {
  static auto get() { return &ln_bwd_kernel<T, P, VEC, TPR, CL>; }
};

// dweight[c], dbias[c] = sum over blocks of partial[b][0 / 1][c]: 32 columns a
// block, 8 strips of block sums added in strip order. Either output may be null.
template <class P>
__global__ void __launch_bounds__(256) ln_param_kernel(const float* __restrict__ partial, int nblk, int d,
                                                       P* __restrict__ dweight, P* __restrict__ dbias) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, strip = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, n = 2 * (int64_t)d;
  float v = 0.0f;
  if (c < n) {
#pragma unroll 8
    for (int b = strip; b < nblk; b += 8) v += partial[b * n + c];
  }
  s[strip][lane] = v;
  __syncthreads();
  if (strip == 0 && c < n) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) t += s[k][lane];
    P* out = c < d ? dweight : dbias;
    if (out) out[c < d ? c : c - d] = from_f32<P>(t);
  }
}

template <class P>
int launch_params(const float* partial, int nblk, int d, void* dw, void* db, cudaStream_t s) {
  ln_param_kernel<P><<<(unsigned)((2 * (int64_t)d + 31) / 32), 256, 0, s>>>(partial, nblk, d, (P*)dw, (P*)db);
  VRS_CUDA(cudaGetLastError());
  count_launch();
  return VRS_OK;
}

}  // namespace
}  // namespace ops
}  // namespace vrs

extern "C" int vrs_layer_norm_backward_workspace(int64_t rows, int64_t d, int64_t* out_bytes) {
  using namespace vrs::ops;
  if (!out_bytes) return invalid("vrs_layer_norm_backward_workspace: null out_bytes");
  VRS_TRY(ln_check("vrs_layer_norm_backward_workspace", rows, d, VRS_F32, VRS_F32));
  int sms = 0;
  VRS_TRY(sm_count(&sms));
  // The plan with and without 16-byte accesses differs in the cluster only,
  // which lowers the block count.
  const LnPlan p = ln_plan(rows, (int)d, kE, 1, false, sms, kBlocksPerSm);
  const LnPlan q = ln_plan(rows, (int)d, kE, 8, true, sms, kBlocksPerSm);
  *out_bytes = (int64_t)(p.blocks > q.blocks ? p.blocks : q.blocks) * 2 * d * (int64_t)sizeof(float);
  return VRS_OK;
}

extern "C" int vrs_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                       int64_t rows, int64_t d, int32_t dtype, const void* weight,
                                       int32_t param_dtype, const float* mean, const float* rstd, void* dx,
                                       int64_t dx_stride, void* dweight, void* dbias, void* workspace,
                                       int64_t workspace_bytes, void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  VRS_TRY(ln_check("vrs_layer_norm_backward", rows, d, dtype, param_dtype));
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (rows == 0) {  // sums over no rows
    const size_t bytes = (size_t)d * dtype_bytes(param_dtype);
    if (dweight) VRS_CUDA(cudaMemsetAsync(dweight, 0, bytes, s));
    if (dbias) VRS_CUDA(cudaMemsetAsync(dbias, 0, bytes, s));
    return VRS_OK;
  }
  if (!dy || !x || !mean || !rstd || !dx) return invalid("vrs_layer_norm_backward: null buffer");
  if (rows > 1 && (x_stride < d || dy_stride < d || dx_stride < d))
    return invalid("vrs_layer_norm_backward: row strides must be at least d");
  const int vec = 16 / dtype_bytes(dtype);
  const bool can_vec = d % vec == 0 &&
                       (rows == 1 || (x_stride % vec == 0 && dy_stride % vec == 0 && dx_stride % vec == 0)) &&
                       aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(weight);
  int sms = 0;
  VRS_TRY(sm_count(&sms));
  const LnPlan p = ln_plan(rows, (int)d, kE, vec, can_vec, sms, kBlocksPerSm);
  const bool params = dweight || dbias;
  if (params) {
    if (!workspace) return invalid("vrs_layer_norm_backward: null workspace");
    if (((uintptr_t)workspace & 3) != 0) return invalid("vrs_layer_norm_backward: workspace must be 4-byte aligned");
    if (workspace_bytes < (int64_t)p.blocks * 2 * d * (int64_t)sizeof(float))
      return invalid("vrs_layer_norm_backward: workspace of " + std::to_string(workspace_bytes) +
                     " bytes is smaller than vrs_layer_norm_backward_workspace says");
  }
  LnArgs a{};
  a.x = x;
  a.dy = dy;
  a.weight = weight;
  a.y = dx;
  a.mean_in = mean;
  a.rstd_in = rstd;
  a.partial = params ? (float*)workspace : nullptr;
  a.rows = rows;
  a.xs = x_stride;
  a.dys = dy_stride;
  a.ys = dx_stride;
  a.d = (int)d;
  ProfToken t = prof_begin("layer_norm_backward", s);
  int st = ln_dispatch<BwdKernel>(dtype, param_dtype, a, p, s);
  if (st == VRS_OK && params) {
    st = param_dtype == VRS_F32   ? launch_params<float>(a.partial, p.blocks, a.d, dweight, dbias, s)
         : param_dtype == VRS_F16 ? launch_params<f16>(a.partial, p.blocks, a.d, dweight, dbias, s)
                                  : launch_params<bf16>(a.partial, p.blocks, a.d, dweight, dbias, s);
  }
  prof_end(t, s);
  return st;
}
