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
//
// The instructions come next after memory (33 an element in a first form kept
// it at 4.2 TB/s): pairs of floats, and two rows to a reduction.
//
// A thread's loads of the next rows are in flight while it reduces the
// current ones: asynchronous copies into slots of its own in shared memory
// (nobody else reads them, so no barrier is added).
//
// Few rows (at most kColumnRows): the blocks' sums would be as large as the
// inputs. Further blocks of the same launch then sum the columns straight
// from x and dy, which L2 still holds.
#include <cuda_pipeline_primitives.h>

#include "layer_norm.cuh"

namespace vrs {
namespace ops {
namespace {

// Elements a thread holds of each row it has at a time, and blocks an SM. 8
// (two rows) leave room for 24 warps; 16 reach the widest rows with clusters
// of 8.
constexpr int kNarrow = 8, kWide = 16;
constexpr int kNarrowRows = 2, kWideRows = 1;
constexpr int kNarrowBlocks = 3, kWideBlocks = 2;
constexpr int64_t kColumnRows = 64;
constexpr int kColumns = 64;  // of a column block; its 4 strips of threads split the rows

// Asynchronous copies: bytes of a stage (the rows of one turn), and stages.
template <class T, int E>
constexpr int stage_bytes() {
  return (E == kNarrow ? kNarrowRows : kWideRows) * 2 * E * (int)sizeof(T) * kLnThreads;
}
template <class T, int E>
constexpr int stage_count() {
  return stage_bytes<T, E>() <= 16384 ? 3 : 2;
}

template <class T, class P>
__device__ void sum_columns(const LnArgs& a, int block, float (*s)[kColumns][2]) {
  const T* x = (const T*)a.x;
  const T* dy = (const T*)a.dy;
  const int lane = threadIdx.x % kColumns, strip = threadIdx.x / kColumns;
  const int c = block * kColumns + lane;
  float dw = 0.0f, db = 0.0f;
  if (c < a.d) {
#pragma unroll 8
    for (int r = strip; r < (int)a.rows; r += kLnThreads / kColumns) {
      const float g = to_f32(dy[r * a.dys + c]);
      dw = fmaf(g, (to_f32(x[r * a.xs + c]) - a.mean_in[r]) * a.rstd_in[r], dw);
      db += g;
    }
  }
  s[strip][lane][0] = dw;
  s[strip][lane][1] = db;
  __syncthreads();
  if (strip == 0 && c < a.d) {
#pragma unroll
    for (int k = 1; k < kLnThreads / kColumns; k++) {
      dw += s[k][lane][0];
      db += s[k][lane][1];
    }
    if (a.dweight) ((P*)a.dweight)[c] = from_f32<P>(dw);
    if (a.dbias) ((P*)a.dbias)[c] = from_f32<P>(db);
  }
}

template <class T, class P, int VEC, int TPR, int E, bool CL>
__global__ void __launch_bounds__(kLnThreads, E == kNarrow ? kNarrowBlocks : kWideBlocks)
    ln_bwd_kernel(const LnArgs a) {
  constexpr int NV = E / VEC, GROUPS = kLnThreads / TPR, R = E == kNarrow ? kNarrowRows : kWideRows;
  constexpr bool ASYNC = VEC > 1;
  constexpr int DEPTH = stage_count<T, E>();
  using Red = LnReduce<TPR, CL, 2 * R>;
  __shared__ typename Red::Smem s_red;
  constexpr int kColFloats = GROUPS > 1 ? 2 * TPR * E : kLnThreads * 2;
  __shared__ float s_col[kColFloats];
  extern __shared__ uint4 s_row[];  // ASYNC: [DEPTH][R][2][NV][threads]
  int64_t first = blockIdx.x, step = gridDim.x - a.col_blocks;
  if (first >= step) {  // whole clusters
    sum_columns<T, P>(a, (int)(first - step), reinterpret_cast<float(*)[kColumns][2]>(s_col));
    return;
  }
  int tt = threadIdx.x % TPR, TT = TPR;
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
  const float inv_d = 1.0f / (float)a.d;
  const int64_t turn = step * (GROUPS * R);
  const int64_t row0 = first * (GROUPS * R) + threadIdx.x / TPR;  // and every GROUPS-th after it

  auto slot_of = [&](int at, int r, int which, int i) {
    return &s_row[(((at * R + r) * 2 + which) * NV + i) * kLnThreads + threadIdx.x];
  };
  auto fetch = [&](int64_t row, int at) {
    if constexpr (ASYNC) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        if (row + r * GROUPS < a.rows) {
          const T* px = x + (row + r * GROUPS) * a.xs;
          const T* py = dy + (row + r * GROUPS) * a.dys;
#pragma unroll
          for (int i = 0; i < NV; i++) {
            const int c = (i * TT + tt) * VEC;
            if (c < a.d) {
              __pipeline_memcpy_async(slot_of(at, r, 0, i), px + c, 16);
              __pipeline_memcpy_async(slot_of(at, r, 1, i), py + c, 16);
            }
          }
        }
      }
      __pipeline_commit();
    }
  };
  if constexpr (ASYNC) {
    // Columns past the row's end are zeros and stay so.
#pragma unroll
    for (int i = 0; i < NV; i++)
      if ((i * TT + tt) * VEC >= a.d)
        for (int k = 0; k < DEPTH * R * 2; k++) *slot_of(k / (R * 2), k / 2 % R, k % 2, i) = make_uint4(0, 0, 0, 0);
    for (int k = 0; k < DEPTH - 1; k++) fetch(row0 + k * turn, k);
  }

  Held<P, E, VEC> w;
  w.fill(1.0f);
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int c = (i * TT + tt) * VEC;
    if (a.weight && c < a.d) w.load(i, (const P*)a.weight + c);
  }
  F2 dw[E / 2], db[E / 2];
#pragma unroll
  for (int q = 0; q < E / 2; q++) dw[q] = db[q] = pack_f2(0.0f);
  int slot = 0, at = 0;
  // Every thread of a block takes the same number of turns; a row past the
  // last one is zeros (with dy = 0 it adds nothing to any sum).
  for (int64_t row = row0, r0 = first * (GROUPS * R); r0 < a.rows; row += turn, r0 += turn) {
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const bool have = row + r * GROUPS < a.rows;
      mean[r] = have ? a.mean_in[row + r * GROUPS] : 0.0f;
      rstd[r] = have ? a.rstd_in[row + r * GROUPS] : 0.0f;
    }
    if constexpr (ASYNC) {
      fetch(row + (DEPTH - 1) * turn, at == 0 ? DEPTH - 1 : at - 1);
      __pipeline_wait_prior(DEPTH - 1);
    }
    F2 xh[R][E / 2], g[R][E / 2];
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const bool have = row + r * GROUPS < a.rows;
      Held<T, E, VEC> kx, ky;
      kx.fill(0.0f);
      ky.fill(0.0f);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int c = (i * TT + tt) * VEC;
        if constexpr (ASYNC) {
          if (have) {
            kx.k[i] = *reinterpret_cast<const Pack<T, VEC>*>(slot_of(at, r, 0, i));
            ky.k[i] = *reinterpret_cast<const Pack<T, VEC>*>(slot_of(at, r, 1, i));
          }
        } else if (have && c < a.d) {
          kx.load(i, x + (row + r * GROUPS) * a.xs + c);
          ky.load(i, dy + (row + r * GROUPS) * a.dys + c);
        }
      }
      const F2 m = pack_f2(-mean[r]), f = pack_f2(rstd[r]);
      F2 s0 = pack_f2(0.0f), s1 = pack_f2(0.0f);
#pragma unroll
      for (int q = 0; q < E / 2; q++) {
        const F2 d_y = ky.pair(q);
        xh[r][q] = mul2(add2(kx.pair(q), m), f);
        dw[q] = fma2(d_y, xh[r][q], dw[q]);
        db[q] = add2(db[q], d_y);
        g[r][q] = mul2(d_y, w.pair(q));
        s0 = add2(s0, g[r][q]);
        s1 = fma2(g[r][q], xh[r][q], s1);
      }
      s[2 * r] = sum_f2(s0);
      s[2 * r + 1] = sum_f2(s1);
    }
    if constexpr (ASYNC) at = at + 1 == DEPTH ? 0 : at + 1;
    Red::run(s, &s_red, slot);
    slot ^= 1;
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (row + r * GROUPS >= a.rows) break;
      const F2 f = pack_f2(rstd[r]), m0 = pack_f2(-s[2 * r] * inv_d), m1 = pack_f2(-s[2 * r + 1] * inv_d);
#pragma unroll
      for (int q = 0; q < E / 2; q++) g[r][q] = mul2(add2(g[r][q], fma2(xh[r][q], m1, m0)), f);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int c = (i * TT + tt) * VEC;
        if (c < a.d) store_held<T, VEC, E>(dx + (row + r * GROUPS) * a.ys + c, g[r], i);
      }
    }
  }
  if constexpr (ASYNC) __pipeline_wait_prior(0);
  if (a.partial) {
    float* out = a.partial + first * 2 * a.d;
    float fw[E], fb[E];
#pragma unroll
    for (int q = 0; q < E / 2; q++) {
      unpack_f2(dw[q], fw[2 * q], fw[2 * q + 1]);
      unpack_f2(db[q], fb[2 * q], fb[2 * q + 1]);
    }
    if constexpr (GROUPS > 1) {
      // The groups of a block add their sums in turn (always in this order).
      for (int gr = 0; gr < GROUPS; gr++) {
        if ((int)threadIdx.x / TPR == gr) {
#pragma unroll
          for (int e = 0; e < E; e++) {
            const int c = (e / VEC * TT + tt) * VEC + e % VEC;
            if (c < a.d) {
              s_col[c] = (gr ? s_col[c] : 0.0f) + fw[e];
              s_col[TPR * E + c] = (gr ? s_col[TPR * E + c] : 0.0f) + fb[e];
            }
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < a.d; c += kLnThreads) {
        out[c] = s_col[c];
        out[a.d + c] = s_col[TPR * E + c];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int c = (e / VEC * TT + tt) * VEC + e % VEC;
        if (c < a.d) {
          out[c] = fw[e];
          out[a.d + c] = fb[e];
        }
      }
    }
  }
  // A block must not leave while another still writes its shared memory.
  if constexpr (CL) cooperative_groups::this_cluster().sync();
}

template <class T, class P, int VEC, int TPR, int E, bool CL>
struct BwdKernel {
  static auto get() { return &ln_bwd_kernel<T, P, VEC, TPR, E, CL>; }
  static int smem() { return VEC > 1 ? stage_count<T, E>() * stage_bytes<T, E>() : 0; }
};

LnPlan bwd_plan(int64_t rows, int d, int vec, bool can_vec, int sms) {
  return ln_plan(rows, d, kNarrow, kWide, kNarrowRows, kWideRows, vec, can_vec, sms, kNarrowBlocks, kWideBlocks);
}

// dweight[c], dbias[c] = sum over blocks of partial[b][0 / 1][c]: 32 columns a
// block, 32 strips of block sums added in strip order (a strip of 444 blocks
// is 14 loads). Either output may be null.
constexpr int kStrips = 32;
template <class P>
__global__ void __launch_bounds__(32 * kStrips) ln_param_kernel(const float* __restrict__ partial, int nblk, int d,
                                                       P* __restrict__ dweight, P* __restrict__ dbias) {
  __shared__ float s[kStrips][33];
  const int lane = threadIdx.x & 31, strip = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, n = 2 * (int64_t)d;
  float v = 0.0f;
  if (c < n) {
#pragma unroll 14
    for (int b = strip; b < nblk; b += kStrips) v += partial[b * n + c];
  }
  s[strip][lane] = v;
  __syncthreads();
  if (strip == 0 && c < n) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < kStrips; k++) t += s[k][lane];
    P* out = c < d ? dweight : dbias;
    if (out) out[c < d ? c : c - d] = from_f32<P>(t);
  }
}

template <class P>
int launch_params(const float* partial, int nblk, int d, void* dw, void* db, cudaStream_t s) {
  ln_param_kernel<P><<<(unsigned)((2 * (int64_t)d + 31) / 32), 32 * kStrips, 0, s>>>(partial, nblk, d, (P*)dw, (P*)db);
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
  const LnPlan p = bwd_plan(rows, (int)d, 1, false, sms);
  const LnPlan q = bwd_plan(rows, (int)d, 8, true, sms);
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
  const LnPlan p = bwd_plan(rows, (int)d, vec, can_vec, sms);
  const bool params = dweight || dbias;
  const bool columns = params && rows <= kColumnRows;
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
  a.partial = params && !columns ? (float*)workspace : nullptr;
  if (columns) {
    a.dweight = dweight;
    a.dbias = dbias;
    a.col_blocks = (int)((d + kColumns - 1) / kColumns + p.cluster - 1) / p.cluster * p.cluster;
  }
  a.rows = rows;
  a.xs = x_stride;
  a.dys = dy_stride;
  a.ys = dx_stride;
  a.d = (int)d;
  ProfToken t = prof_begin("layer_norm_backward", s);
  int st = ln_dispatch<BwdKernel, kNarrow, kWide>(dtype, param_dtype, a, p, s);
  if (st == VRS_OK && a.partial) {
    st = param_dtype == VRS_F32   ? launch_params<float>(a.partial, p.blocks, a.d, dweight, dbias, s)
         : param_dtype == VRS_F16 ? launch_params<f16>(a.partial, p.blocks, a.d, dweight, dbias, s)
                                  : launch_params<bf16>(a.partial, p.blocks, a.d, dweight, dbias, s);
  }
  prof_end(t, s);
  return st;
}
