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
// it at 4.2 TB/s): pairs of floats, and shuffles that halve the values.
//
// Few rows (at most kColumnRows): the blocks' sums would be as large as the
// inputs. Further blocks of the same launch then sum the columns straight
// from x and dy, which L2 still holds.
#include "layer_norm.cuh"

namespace vrs {
namespace ops {
namespace {

// x, dy, the weight and two column sums an element: 16 elements a thread
// leave room for two blocks an SM. (Measured at 65,536 x 2,048 in bf16: 144 us;
// 8 elements, two rows a turn and three blocks 167 us, four blocks 209 us.)
constexpr int kBlocksPerSm = 2;
constexpr int64_t kColumnRows = 64;
constexpr int kColumns = 64;  // of a column block; its 4 strips of threads split the rows

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

template <class T, class P, int VEC, int TPR, int E, int R, bool CL>
__global__ void __launch_bounds__(kLnThreads, kBlocksPerSm)
    ln_bwd_kernel(const LnArgs a) {
  constexpr int GROUPS = kLnThreads / TPR;
  using Ring = LnRing<T, VEC, E, R, 2, CL>;
  using Red = LnReduce<TPR, CL, 2 * R>;
  __shared__ typename Red::Smem s_red;
  // Sums of the block's columns, or of a column block's strips.
  constexpr int kColFloats = GROUPS > 1 && TPR * E > kLnThreads ? 2 * TPR * E : 2 * kLnThreads;
  __shared__ float s_col[kColFloats];
  int64_t first = blockIdx.x, step = gridDim.x - a.col_blocks;
  grid_launch();
  grid_wait();
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
  T* dx = (T*)a.y;
  const float inv_d = 1.0f / (float)a.d;
  const int64_t apart = step * GROUPS;
  LnPlace<VEC> at;
  at.tt = tt;
  at.TT = TT;
  const int64_t row0 = at.start(a, first, GROUPS, threadIdx.x / TPR);
  Ring ring;
  ring.base[0] = (const T*)a.x;
  ring.base[1] = (const T*)a.dy;
  ring.stride[0] = a.xs;
  ring.stride[1] = a.dys;
  ring.rows = a.rows;
  ring.apart = apart;
  ring.at_columns = at;
  ring.start(row0);
  Red::start(&s_red);

  Held<P, E, VEC> w;
  w.fill(1.0f);
  at.load(w, a.weight);
  F2 dw[E / 2], db[E / 2];
#pragma unroll
  for (int q = 0; q < E / 2; q++) dw[q] = db[q] = pack_f2(0.0f);
  // A turn's statistics are loaded a turn ahead.
  float mean_next[R], rstd_next[R];
  auto stats = [&](int64_t row) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      const bool have = row + r * apart < a.rows;
      mean_next[r] = have ? a.mean_in[row + r * apart] : 0.0f;
      rstd_next[r] = have ? a.rstd_in[row + r * apart] : 0.0f;
    }
  };
  stats(row0);
  int turn = 0;
  // Every thread of a block takes the same number of turns; a row past the
  // last one is zeros (with dy = 0 it adds nothing to any sum).
  for (int64_t row = row0, r0 = at.first; r0 < a.rows; row += R * apart, r0 += R * apart) {
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      mean[r] = mean_next[r];
      rstd[r] = rstd_next[r];
    }
    stats(row + R * apart);
    ring.next(row);
    F2 xh[R][E / 2], g[R][E / 2];
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const Held<T, E, VEC> kx = ring.get(row, r, 0), ky = ring.get(row, r, 1);
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
    ring.done();
    Red::run(s, &s_red, turn++, a.err);
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (row + r * apart >= a.rows) break;
      const F2 f = pack_f2(rstd[r]), m0 = pack_f2(-s[2 * r] * inv_d), m1 = pack_f2(-s[2 * r + 1] * inv_d);
#pragma unroll
      for (int q = 0; q < E / 2; q++) g[r][q] = mul2(add2(g[r][q], fma2(xh[r][q], m1, m0)), f);
      at.template store<T, E>(dx + (row + r * apart) * a.ys, g[r]);
    }
  }
  ring.drain();
  if (a.partial) {
    float* out = a.partial + first * 2 * a.d;
    float fw[E], fb[E];
#pragma unroll
    for (int q = 0; q < E / 2; q++) {
      unpack_f2(dw[q], fw[2 * q], fw[2 * q + 1]);
      unpack_f2(db[q], fb[2 * q], fb[2 * q + 1]);
    }
    if constexpr (TPR < 32) {
#pragma unroll
      for (int o = TPR; o < 32; o *= 2)
#pragma unroll
        for (int e = 0; e < E; e++) {
          fw[e] += __shfl_xor_sync(0xffffffffu, fw[e], o);
          fb[e] += __shfl_xor_sync(0xffffffffu, fb[e], o);
        }
    }
    if constexpr (GROUPS > 1) {
      // The groups of a block (warps, where a row takes less) add their sums
      // in turn, always in this order.
      constexpr int SPAN = TPR < 32 ? 32 : TPR;
      for (int gr = 0; gr < kLnThreads / SPAN; gr++) {
        if ((int)threadIdx.x / SPAN == gr && (int)threadIdx.x % SPAN < TPR) {
#pragma unroll
          for (int e = 0; e < E; e++) {
            const int c = at.column(e / VEC) + e % VEC;
            if (at.has(e / VEC, e % VEC)) {
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
        const int c = at.column(e / VEC) + e % VEC;
        if (at.has(e / VEC, e % VEC)) {
          out[c] = fw[e];
          out[a.d + c] = fb[e];
        }
      }
    }
  }
  // A block must not leave while another still writes its shared memory.
  if constexpr (CL) cooperative_groups::this_cluster().sync();
}

template <class T, class P, int VEC, int TPR, int E, int R, bool CL>
struct BwdKernel {
  static auto get() { return &ln_bwd_kernel<T, P, VEC, TPR, E, R, CL>; }
  static int smem() {
    return LnRing<T, VEC, E, R, 2, CL>::kBytes;
  }
};

LnPlan bwd_plan(int64_t rows, int d, int vec, LnAccess access, int sms) {
  return ln_plan(rows, d, false, vec, access, sms, kBlocksPerSm);
}

// dweight[c], dbias[c] = sum over blocks of partial[b][0 / 1][c]: 32 columns a
// block, 32 strips of block sums added in strip order (a strip of 444 blocks
// is 14 loads). Either output may be null.
constexpr int kStrips = 32;
template <class P>
__global__ void __launch_bounds__(32 * kStrips) ln_param_kernel(const float* __restrict__ partial, int nblk, int d,
                                                       P* __restrict__ dweight, P* __restrict__ dbias) {
  __shared__ float s[kStrips][33];
  grid_launch();
  grid_wait();
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
  VRS_TRY(launch_after(ln_param_kernel<P>, (unsigned)((2 * (int64_t)d + 31) / 32), 32 * kStrips, 0, s, partial, nblk, d,
                       (P*)dw, (P*)db));
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
  // How the rows can be reached decides the cluster of few rows and whether
  // the count of blocks is even. Rows in wider clusters have fewer of them, and so
  // may more rows than SMs: the answer is the largest of all widths up to d and of
  // both counts of rows, so that a workspace for the largest sizes serves all
  // smaller ones.
  auto bytes = [&](int64_t width) {
    int blocks = 0;
    for (int64_t n : {rows, rows < sms ? rows : (int64_t)sms})
      for (LnAccess access : {kLnElements, kLn16Bytes, kLnPairs}) {
        const LnPlan p = bwd_plan(n, (int)width, 8, access, sms);
        blocks = blocks > p.blocks ? blocks : p.blocks;
      }
    return (int64_t)((blocks + 1) / 2 * 2) * 2 * width * (int64_t)sizeof(float);
  };
  constexpr int64_t kOne = kLnThreads * kNarrowE;  // elements that a block of a cluster holds
  int64_t most = bytes(d);
  for (int64_t w = kOne; w < d; w += kOne) {
    const int64_t b = bytes(w);
    most = most > b ? most : b;
  }
  *out_bytes = most;
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
  const int bytes = dtype_bytes(dtype);
  const LnRows arrays[] = {{x, x_stride}, {dy, dy_stride}, {dx, dx_stride}};
  const LnAccess access = ln_access(arrays, rows, d, bytes, aligned16(weight));
  int sms = 0;
  VRS_TRY(sm_count(&sms));
  LnPlan p = bwd_plan(rows, (int)d, 16 / bytes, access, sms);
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
  VRS_TRY(error_word(&a.err));
  ProfToken t = prof_begin("layer_norm_backward", s);
  int st = ln_dispatch<BwdKernel, false>(dtype, param_dtype, a, p, s);
  if (st == VRS_OK && a.partial) {
    st = param_dtype == VRS_F32   ? launch_params<float>(a.partial, p.blocks, a.d, dweight, dbias, s)
         : param_dtype == VRS_F16 ? launch_params<f16>(a.partial, p.blocks, a.d, dweight, dbias, s)
                                  : launch_params<bf16>(a.partial, p.blocks, a.d, dweight, dbias, s);
  }
  prof_end(t, s);
  return st;
}
