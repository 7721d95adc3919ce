// layer_norm_fwd.cu -- y = (x - mean) * rstd * weight + bias over rows, with
// mean and rstd = 1 / sqrt(var + eps) kept in 32 bits for the backward pass.
//
// Bound by memory: 2 d elements a row. The row stays in registers between the
// two sums (mean first, then the squares of x - mean: one pass of
// sum-of-squares would lose the variance of rows whose mean is large).
#include "layer_norm.cuh"

namespace vrs {
namespace ops {
namespace {

constexpr int blocks_per_sm(int e) { return e == kWideE ? 2 : e == kBetweenE ? kBetweenBlocks : 3; }

template <class T, class P, int VEC, int TPR, int E, int R, bool CL>
__global__ void __launch_bounds__(kLnThreads, blocks_per_sm(E))
    ln_fwd_kernel(const LnArgs a) {
  constexpr int GROUPS = kLnThreads / TPR;
  using Red = LnReduce<TPR, CL, R>;
  using Ring = LnRing<T, VEC, E, R, 1, CL>;
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
  grid_launch();
  grid_wait();
  T* y = (T*)a.y;
  const int64_t apart = step * GROUPS;
  LnPlace<VEC> at;
  at.tt = tt;
  at.TT = TT;
  const int64_t row_first = at.start(a, first, GROUPS, threadIdx.x / TPR);
  Ring ring;
  ring.base[0] = (const T*)a.x;
  ring.stride[0] = a.xs;
  ring.rows = a.rows;
  ring.apart = apart;
  ring.at_columns = at;
  ring.start(row_first);
  Red::start(&s_red);
  const float inv_d = 1.0f / (float)a.d;
  // The parameters of the thread's columns stay in registers for all rows;
  // without them 1 and 0 give the same bits as leaving the steps out (but for
  // the sign of a zero).
  Held<P, E, VEC> w, b;
  w.fill(1.0f);
  b.fill(0.0f);
  at.load(w, a.weight);
  at.load(b, a.bias);
  int turn = 0;
  // Every thread of a block takes the same number of turns (the barriers
  // inside the reductions); a group past the last row computes on zeros.
  for (int64_t row0 = row_first, r0 = at.first; r0 < a.rows; row0 += R * apart, r0 += R * apart) {
    ring.next(row0);
    F2 v[R][E / 2];
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const Held<T, E, VEC> k = ring.get(row0, r, 0);
      F2 s = pack_f2(0.0f);
#pragma unroll
      for (int q = 0; q < E / 2; q++) s = add2(s, v[r][q] = k.pair(q));
      mean[r] = sum_f2(s);
    }
    ring.done();
    Red::run(mean, &s_red, turn++, a.err);
#pragma unroll
    for (int r = 0; r < R; r++) {
      mean[r] *= inv_d;
      const F2 m = pack_f2(-mean[r]);
      F2 s = pack_f2(0.0f);
#pragma unroll
      for (int q = 0; q < E / 2; q++) {
        v[r][q] = add2(v[r][q], m);
        if constexpr (VEC > 2) {
          if (at.column(2 * q / VEC) < a.d) s = fma2(v[r][q], v[r][q], s);
        } else {
          float lo, hi;
          unpack_f2(v[r][q], lo, hi);
          const F2 in = pack_f2(at.has(2 * q / VEC, 2 * q % VEC) ? lo : 0.0f,
                                at.has((2 * q + 1) / VEC, (2 * q + 1) % VEC) ? hi : 0.0f);
          s = fma2(in, in, s);
        }
      }
      rstd[r] = sum_f2(s);
    }
    Red::run(rstd, &s_red, turn++, a.err);
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int64_t row = row0 + r * apart;
      if (row >= a.rows) break;
      rstd[r] = 1.0f / sqrtf(fmaf(rstd[r], inv_d, a.eps));
      if (tt == 0) {
        if (a.mean) a.mean[row] = mean[r];
        if (a.rstd) a.rstd[row] = rstd[r];
      }
      const F2 f = pack_f2(rstd[r]);
#pragma unroll
      for (int q = 0; q < E / 2; q++) v[r][q] = fma2(mul2(v[r][q], f), w.pair(q), b.pair(q));
      at.template store<T, E>(y + row * a.ys, v[r]);
    }
  }
  ring.drain();
  // A block must not leave while another still writes its shared memory.
  if constexpr (CL) cooperative_groups::this_cluster().sync();
}

template <class T, class P, int VEC, int TPR, int E, int R, bool CL>
struct FwdKernel {
  static auto get() { return &ln_fwd_kernel<T, P, VEC, TPR, E, R, CL>; }
  static int smem() {
    return LnRing<T, VEC, E, R, 1, CL>::kBytes;
  }
};

}  // namespace

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
  const int bytes = dtype_bytes(dtype);
  const LnRows arrays[] = {{x, x_stride}, {y, y_stride}};
  const LnAccess access = ln_access(arrays, rows, d, bytes, aligned16(weight) && aligned16(bias));
  int sms = 0;
  VRS_TRY(sm_count(&sms));
  VRS_TRY(error_word(&a.err));
  LnPlan p = ln_plan(rows, (int)d, true, 16 / bytes, access, sms, blocks_per_sm(d > kLnThreads * kNarrowE ? kWideE : 0));
  cudaStream_t s = (cudaStream_t)cuda_stream;
  ProfToken t = prof_begin("layer_norm_forward", s);
  const int st = ln_dispatch<FwdKernel, true>(dtype, param_dtype, a, p, s);
  prof_end(t, s);
  return st;
}
