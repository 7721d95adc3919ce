// qk_norm_rope.cu -- the RMS norm of each head's query and key with the
// rotation to its position, and their gradients:
//   xhat = x rstd, rstd = 1 / sqrt(mean x^2 + eps), u = xhat w,
//   y = u but for the pairs of the first `rotary` elements, turned by
//   position * base^(-2 i / rotary): (a cos - b sin, b cos + a sin).
// Backward g is dy turned back (the rotation's transpose), dw = sum g xhat,
// dx = rstd (g w - xhat mean(g w xhat)). rstd is computed again from x: it costs
// no reading, since dw needs x.
//
// Bound by memory: a head in and out (backward two in, one out). A group of 1 to
// 32 lanes holds a head in registers, as pairs: each lane has V neighbouring
// pairs, read as two accesses of V elements. A warp takes one token's heads in
// turn; the pairs of a lane, and so its cosines, sines and weights, are the same
// for all of them.
//
// Angles: position times frequency in 64 bits, in turns, of which the whole ones
// are dropped before the sine is taken in 32 bits: positions of millions turn
// the fastest pair by as many radians, of which 32 bits would leave two digits.
#include <cmath>

#include "ops_common.cuh"

namespace vrs {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMostD = 256;
constexpr int kMostBlocks = 148 * 6;   // of the backward pass: partial sums of the weights' gradients
constexpr int kFinishRows = 32;        // threads that share a column of those

struct Heads {
  const void* x;
  int64_t stride, head;  // in elements
  int n;
  const void* w;   // null: ones
  void* y;         // packed
  const void* dy;  // backward
  int64_t dstride, dhead;
};

struct RopeArgs {
  Heads q, k;
  int64_t tokens;
  int d, rotary;
  float eps, inv_d;
  const int64_t* pos;
  int splits, per;  // a token's heads are split for `splits` warps, `per` each
  float* partial;   // [blocks][2][d]
  double turns[kMostD / 2];  // turns a position of each pair
};

// V pairs of a lane: where their elements lie and what turns them.
template <int V, bool INTER>
struct Slot {
  int a, b;   // elements of the two accesses; -1: none
  int first;  // pair
};

template <int V, bool INTER>
__device__ __forceinline__ Slot<V, INTER> slot_of(const RopeArgs& a, int slot) {
  Slot<V, INTER> s;
  const int p = slot * V, half = a.rotary / 2;
  s.first = p;
  if (p >= a.d / 2) {
    s.a = s.b = -1;
  } else if (INTER || p >= half) {  // neighbours (the elements that are not turned too)
    s.a = 2 * p;
    s.b = 2 * p + V;
  } else {
    s.a = p;
    s.b = p + half;
  }
  return s;
}

// One head's pairs of a lane, as floats: e[0..V) from the first access, e[V..2V)
// from the second.
template <class T, int V>
__device__ __forceinline__ void load_slot(const T* p, int a, int b, float (&e)[2 * V]) {
  const Pack<T, V> x = load_pack<T, V>(p + a), y = load_pack<T, V>(p + b);
#pragma unroll
  for (int j = 0; j < V; j++) {
    e[j] = to_f32(x.v[j]);
    e[V + j] = to_f32(y.v[j]);
  }
}

// Turns the pairs by (cos, sin); SIGN -1 turns back. Slots that are not turned
// have cosine 1 and sine 0, which leaves finite values as they are; `turned`
// keeps a 0 times an infinity out of them.
template <int V, bool INTER>
__device__ __forceinline__ void turn(float (&e)[2 * V], const float (&c)[V], const float (&s)[V], float sign, bool turned) {
  if (!turned) return;
#pragma unroll
  for (int j = 0; j < V; j++) {
    float &a = INTER ? e[2 * j] : e[j], &b = INTER ? e[2 * j + 1] : e[V + j];
    const float x = a, y = b, sn = s[j] * sign;
    a = x * c[j] - y * sn;
    b = y * c[j] + x * sn;
  }
}

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// V pairs an access, L lanes a head, S accesses a lane; BACK: the gradients.
template <class T, class P, int V, int L, int S, bool INTER, bool BACK>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 s_turn[kWarps][kMostD / 2];
  __shared__ double s_freq[kMostD / 2];  // (lanes read different ones: constant memory would serve them in turn)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane % L, group = lane / L;
  constexpr int G = 32 / L;  // heads at a time
  for (int p = threadIdx.x; p < a.rotary / 2; p += kThreads) s_freq[p] = a.turns[p];
  __syncthreads();
  grid_launch();
  grid_wait();
  Slot<V, INTER> slot[S];
  float w[2][S][2 * V];   // weights of queries and keys
  float dw[2][S][2 * V];
#pragma unroll
  for (int s = 0; s < S; s++) {
    slot[s] = slot_of<V, INTER>(a, gl + s * L);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const P* from = (const P*)(h ? a.k.w : a.q.w);
#pragma unroll
      for (int j = 0; j < 2 * V; j++) {
        const int at = j < V ? slot[s].a + j : slot[s].b + j - V;
        w[h][s][j] = slot[s].a >= 0 && from ? to_f32(from[at]) : 1.0f;
        dw[h][s][j] = 0.0f;
      }
    }
  }
  const int heads = a.q.n + a.k.n, half = a.rotary / 2;
  const int64_t units = a.tokens * a.splits;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + warp; u < units; u += (int64_t)gridDim.x * kWarps) {
    const int64_t t = u / a.splits;
    const int h0 = (int)(u % a.splits) * a.per, h1 = min(heads, h0 + a.per);
    // The token's cosines and sines, each computed by one lane.
    const double at = half ? (double)a.pos[t] : 0.0;
    __syncwarp();
    for (int p = lane; p < half; p += 32) {
      const double turns = at * s_freq[p];
      float sn, cs;
      sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
      s_turn[warp][p] = make_float2(cs, sn);
    }
    __syncwarp();
    float cs[S][V], sn[S][V];
    bool turned[S];
#pragma unroll
    for (int s = 0; s < S; s++) {
      turned[s] = slot[s].a >= 0 && slot[s].first < half;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float2 f = turned[s] ? s_turn[warp][slot[s].first + j] : make_float2(1.0f, 0.0f);
        cs[s][j] = f.x;
        sn[s][j] = f.y;
      }
    }
#pragma unroll 2
    for (int i = h0; i < h1; i += G) {
      const int head = i + group;
      const bool live = head < h1, key = head >= a.q.n;
      const int h = key ? head - a.q.n : head;
      const T* x = (const T*)(key ? a.k.x : a.q.x) + t * (key ? a.k.stride : a.q.stride) + h * (key ? a.k.head : a.q.head);
      T* y = (T*)(key ? a.k.y : a.q.y) + (t * (key ? a.k.n : a.q.n) + h) * a.d;
      float e[S][2 * V], g[S][2 * V];
      float sq = 0.0f;
#pragma unroll
      for (int s = 0; s < S; s++) {
#pragma unroll
        for (int j = 0; j < 2 * V; j++) e[s][j] = g[s][j] = 0.0f;
        if (live && slot[s].a >= 0) {
          load_slot<T, V>(x, slot[s].a, slot[s].b, e[s]);
          if (BACK) {
            const T* dy = (const T*)(key ? a.k.dy : a.q.dy) + t * (key ? a.k.dstride : a.q.dstride) +
                          h * (key ? a.k.dhead : a.q.dhead);
            load_slot<T, V>(dy, slot[s].a, slot[s].b, g[s]);
          }
        }
#pragma unroll
        for (int j = 0; j < 2 * V; j++) sq = fmaf(e[s][j], e[s][j], sq);
      }
      sq = group_sum<L>(sq);
      const float rstd = 1.0f / sqrtf(sq * a.inv_d + a.eps);
      if (BACK) {
        float mean = 0.0f;
#pragma unroll
        for (int s = 0; s < S; s++) {
          turn<V, INTER>(g[s], cs[s], sn[s], -1.0f, turned[s]);
#pragma unroll
          for (int j = 0; j < 2 * V; j++) {
            e[s][j] *= rstd;
            const float f = g[s][j] * e[s][j];
            // (A select, so that each thread's sums stay in registers.)
            dw[0][s][j] += live && !key ? f : 0.0f;
            dw[1][s][j] += live && key ? f : 0.0f;
            g[s][j] *= key ? w[1][s][j] : w[0][s][j];
            mean = fmaf(g[s][j], e[s][j], mean);
          }
        }
        mean = group_sum<L>(mean) * a.inv_d;
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
          for (int j = 0; j < 2 * V; j++) e[s][j] = (g[s][j] - e[s][j] * mean) * rstd;
      } else {
#pragma unroll
        for (int s = 0; s < S; s++) {
#pragma unroll
          for (int j = 0; j < 2 * V; j++) e[s][j] = e[s][j] * rstd * (key ? w[1][s][j] : w[0][s][j]);
          turn<V, INTER>(e[s], cs[s], sn[s], 1.0f, turned[s]);
        }
      }
#pragma unroll
      for (int s = 0; s < S; s++)
        if (live && slot[s].a >= 0) {
          store_pack<T, V>(y + slot[s].a, &e[s][0]);
          store_pack<T, V>(y + slot[s].b, &e[s][V]);
        }
    }
  }
  if (!BACK || !a.partial) return;
  // The block's sums for each column, its groups' in order.
  __shared__ float s_dw[kWarps][kMostD];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int j = 0; j < 2 * V; j++) {
        float v = dw[h][s][j];
#pragma unroll
        for (int o = L; o < 32; o <<= 1) v += __shfl_xor_sync(~0u, v, o);
        if (group == 0 && slot[s].a >= 0) s_dw[warp][j < V ? slot[s].a + j : slot[s].b + j - V] = v;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += kThreads) {
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps; i++) v += s_dw[i][c];
      a.partial[((int64_t)blockIdx.x * 2 + h) * a.d + c] = v;
    }
  }
}

// dweight[c] = sum over blocks of partial[block][h][c], in order: 8 columns a
// block, 32 threads a column, each every 32nd block.
template <class P>
__global__ void __launch_bounds__(256) qk_norm_rope_finish_kernel(const float* partial, int blocks, int d, P* dqw, P* dkw) {
  __shared__ float s[kFinishRows][9];
  grid_launch();
  grid_wait();
  const int c = blockIdx.x * 8 + (threadIdx.x & 7), r = threadIdx.x >> 3;
  float v = 0.0f;
  if (c < 2 * d)
    for (int b = r; b < blocks; b += kFinishRows) v += partial[(int64_t)b * 2 * d + c];
  s[r][threadIdx.x & 7] = v;
  __syncthreads();
  if (r == 0 && c < 2 * d) {
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kFinishRows; i++) v += s[i][threadIdx.x & 7];
    P* to = c < d ? dqw : dkw;
    if (to) to[c < d ? c : c - d] = from_f32<P>(v);
  }
}

template <class T, class P, int V, int L, int S, bool INTER, bool BACK>
int launch(RopeArgs& a, int sms, cudaStream_t s, int* blocks) {
  const int heads = a.q.n + a.k.n, at_once = 32 / L;
  // A warp takes all heads of a token where tokens are enough to fill the
  // device (cosines and sines are computed once a token), fewer otherwise.
  const int64_t fill = (int64_t)sms * 4 * kWarps;
  const int turns = (heads + at_once - 1) / at_once;
  const int64_t splits = a.tokens >= fill ? 1 : (fill + a.tokens - 1) / a.tokens;
  const int per = (int)((turns + splits - 1) / splits > 0 ? (turns + splits - 1) / splits : 1);
  a.per = per * at_once;
  a.splits = (heads + a.per - 1) / a.per;
  int64_t grid = (a.tokens * a.splits + kWarps - 1) / kWarps;
  const int64_t most = BACK ? kMostBlocks : (int64_t)sms * 32;
  if (grid > most) grid = most;
  *blocks = (int)grid;
  VRS_TRY(launch_after(qk_norm_rope_kernel<T, P, V, L, S, INTER, BACK>, (unsigned)grid, kThreads, 0, s, a));
  count_launch();
  return VRS_OK;
}

template <class T, class P, int V, bool INTER, bool BACK>
int by_lanes(RopeArgs& a, int sms, cudaStream_t s, int* blocks) {
  const int slots = (a.d / 2 + V - 1) / V;
  if (slots <= 8) return launch<T, P, V, 8, 1, INTER, BACK>(a, sms, s, blocks);
  if (slots <= 16) return launch<T, P, V, 16, 1, INTER, BACK>(a, sms, s, blocks);
  if (slots <= 32) return launch<T, P, V, 32, 1, INTER, BACK>(a, sms, s, blocks);
  if constexpr (V <= 2) {
    if (slots <= 64) return launch<T, P, V, 32, 2, INTER, BACK>(a, sms, s, blocks);
    if constexpr (V == 1) return launch<T, P, V, 32, 4, INTER, BACK>(a, sms, s, blocks);
  }
  return invalid("qk_norm_rope: d is too large");  // (checked before)
}

// V pairs an access where everything divides into it: 8 or 16 bytes a lane.
template <class T, class P, bool BACK>
int by_layout(RopeArgs& a, bool interleaved, bool wide, int sms, cudaStream_t s, int* blocks) {
  constexpr int V = sizeof(T) == 2 ? 4 : 2;
  if (wide)
    return interleaved ? by_lanes<T, P, V, true, BACK>(a, sms, s, blocks) : by_lanes<T, P, V, false, BACK>(a, sms, s, blocks);
  return interleaved ? by_lanes<T, P, 1, true, BACK>(a, sms, s, blocks) : by_lanes<T, P, 1, false, BACK>(a, sms, s, blocks);
}

template <bool BACK>
int by_type(RopeArgs& a, int dtype, int param_dtype, bool interleaved, bool wide, int sms, cudaStream_t s, int* blocks) {
  if (dtype == VRS_F32) return by_layout<float, float, BACK>(a, interleaved, wide, sms, s, blocks);
  if (dtype == VRS_F16)
    return param_dtype == VRS_F32 ? by_layout<f16, float, BACK>(a, interleaved, wide, sms, s, blocks)
                                  : by_layout<f16, f16, BACK>(a, interleaved, wide, sms, s, blocks);
  return param_dtype == VRS_F32 ? by_layout<bf16, float, BACK>(a, interleaved, wide, sms, s, blocks)
                                : by_layout<bf16, bf16, BACK>(a, interleaved, wide, sms, s, blocks);
}

// One array: its alignment in elements is at least V in every stride that counts.
bool fits(const void* p, int64_t stride, int64_t head, int64_t tokens, int n, int v, int bytes) {
  return (uintptr_t)p % (v * bytes) == 0 && (tokens <= 1 || stride % v == 0) && (n <= 1 || head % v == 0);
}

struct Call {
  const vrs_heads *q, *k, *dq_out, *dk_out;  // the last two backward
  int64_t heads, kv_heads, tokens, d;
  int32_t dtype;
  const int64_t* positions;
  const void *q_weight, *k_weight;
  int32_t param_dtype;
  double base;
  int64_t rotary;
  int32_t interleaved;
  float eps;
  void *q_out, *k_out;
};

int check(const char* who, const Call& c, bool back) {
  const std::string w(who);
  if (c.dtype < VRS_F32 || c.dtype > VRS_BF16) return invalid(w + ": dtype must be f32, f16 or bf16");
  if (c.param_dtype != c.dtype && c.param_dtype != VRS_F32) return invalid(w + ": weights are in the heads' type or f32");
  if (c.d < 2 || c.d > kMostD || c.d % 2) return invalid(w + ": d must be even and in 2.." + std::to_string(kMostD));
  if (c.rotary < 0 || c.rotary > c.d || c.rotary % 2) return invalid(w + ": rotary must be even and in 0..d");
  if (c.heads < 1 || c.kv_heads < 1 || c.heads > 65536 || c.kv_heads > 65536)
    return invalid(w + ": heads must be in 1..65536");
  if (c.tokens < 0 || c.tokens > (1ll << 31)) return invalid(w + ": tokens must be in 0..2^31");
  if (!(c.base > 0.0) || !(c.base < INFINITY)) return invalid(w + ": base must be positive and finite");
  if (!(c.eps >= 0.0f)) return invalid(w + ": eps must be at least 0");
  if (c.tokens == 0) return VRS_OK;
  if (!c.q || !c.k || !c.q->data || !c.k->data || !c.q_out || !c.k_out || (c.rotary && !c.positions))
    return invalid(w + ": null heads, positions or results");
  if (back && (!c.dq_out || !c.dk_out || !c.dq_out->data || !c.dk_out->data)) return invalid(w + ": null gradients");
  return VRS_OK;
}

RopeArgs args_of(const Call& c, bool back, bool* wide) {
  RopeArgs a{};
  const int bytes = dtype_bytes(c.dtype), v = c.dtype == VRS_F32 ? 2 : 4;
  bool ok = c.d / 2 % v == 0 && c.rotary / 2 % v == 0;
  auto heads = [&](const vrs_heads& x, int64_t n, const void* w, void* y, const vrs_heads* dy) {
    Heads h{x.data, x.stride, x.head_stride, (int)n, w, y, nullptr, 0, 0};
    ok = ok && fits(x.data, x.stride, x.head_stride, c.tokens, (int)n, v, bytes) && (uintptr_t)y % (v * bytes) == 0;
    if (back) {
      h.dy = dy->data;
      h.dstride = dy->stride;
      h.dhead = dy->head_stride;
      ok = ok && fits(dy->data, dy->stride, dy->head_stride, c.tokens, (int)n, v, bytes);
    }
    return h;
  };
  a.q = heads(*c.q, c.heads, c.q_weight, c.q_out, c.dq_out);
  a.k = heads(*c.k, c.kv_heads, c.k_weight, c.k_out, c.dk_out);
  a.tokens = c.tokens;
  a.d = (int)c.d;
  a.rotary = (int)c.rotary;
  a.eps = c.eps;
  a.inv_d = 1.0f / (float)c.d;
  a.pos = c.positions;
  // base^(-2 i / rotary) / 2 pi
  for (int i = 0; i < a.rotary / 2; i++)
    a.turns[i] = std::pow(c.base, -2.0 * i / (double)a.rotary) / 6.283185307179586476925286766559;
  *wide = ok;
  return a;
}

}  // namespace
}  // namespace ops
}  // namespace vrs

extern "C" int vrs_qk_norm_rope_forward(const vrs_heads* q, int64_t heads, const vrs_heads* k, int64_t kv_heads,
                                        int64_t tokens, int64_t d, int32_t dtype, const int64_t* positions,
                                        const void* q_weight, const void* k_weight, int32_t param_dtype, double base,
                                        int64_t rotary, int32_t interleaved, float eps, void* q_out, void* k_out,
                                        void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  const Call c{q,        k,        nullptr,     nullptr, heads,  kv_heads,    tokens, d,     dtype, positions,
               q_weight, k_weight, param_dtype, base,    rotary, interleaved, eps,    q_out, k_out};
  VRS_TRY(check("vrs_qk_norm_rope_forward", c, false));
  if (tokens == 0) return VRS_OK;
  bool wide = false;
  RopeArgs a = args_of(c, false, &wide);
  int sms = 0, blocks = 0;
  VRS_TRY(sm_count(&sms));
  cudaStream_t s = (cudaStream_t)cuda_stream;
  ProfToken t = prof_begin("qk_norm_rope_forward", s);
  const int st = by_type<false>(a, dtype, param_dtype, interleaved != 0, wide, sms, s, &blocks);
  prof_end(t, s);
  return st;
}

extern "C" int vrs_qk_norm_rope_backward_workspace(int64_t tokens, int64_t d, int64_t* out_bytes) {
  using namespace vrs::ops;
  if (tokens < 0 || d < 2 || d > kMostD || !out_bytes)
    return invalid("vrs_qk_norm_rope_backward_workspace: tokens at least 0, d in 2..256, out_bytes not null");
  *out_bytes = (int64_t)kMostBlocks * 2 * d * 4;
  return VRS_OK;
}

extern "C" int vrs_qk_norm_rope_backward(const vrs_heads* dq_out, const vrs_heads* dk_out, const vrs_heads* q,
                                         int64_t heads, const vrs_heads* k, int64_t kv_heads, int64_t tokens, int64_t d,
                                         int32_t dtype, const int64_t* positions, const void* q_weight,
                                         const void* k_weight, int32_t param_dtype, double base, int64_t rotary,
                                         int32_t interleaved, float eps, void* dq, void* dk, void* dq_weight,
                                         void* dk_weight, void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  const char* who = "vrs_qk_norm_rope_backward";
  const Call c{q,        k,        dq_out,      dk_out, heads,  kv_heads,    tokens, d,  dtype, positions,
               q_weight, k_weight, param_dtype, base,   rotary, interleaved, eps,    dq, dk};
  VRS_TRY(check(who, c, true));
  const bool params = dq_weight || dk_weight;
  int64_t need = 0;
  VRS_TRY(vrs_qk_norm_rope_backward_workspace(tokens, d, &need));
  if (params && (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < need))
    return invalid(std::string(who) + ": workspace missing, off 4 bytes or too small");
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (tokens == 0) {
    const size_t bytes = (size_t)d * dtype_bytes(param_dtype);
    if (dq_weight) VRS_CUDA(cudaMemsetAsync(dq_weight, 0, bytes, s));
    if (dk_weight) VRS_CUDA(cudaMemsetAsync(dk_weight, 0, bytes, s));
    return VRS_OK;
  }
  bool wide = false;
  RopeArgs a = args_of(c, true, &wide);
  a.partial = params ? (float*)workspace : nullptr;
  int sms = 0, blocks = 0;
  VRS_TRY(sm_count(&sms));
  ProfToken t = prof_begin("qk_norm_rope_backward", s);
  int st = by_type<true>(a, dtype, param_dtype, interleaved != 0, wide, sms, s, &blocks);
  if (st == VRS_OK && params) {
    const unsigned grid = (unsigned)((2 * d + 7) / 8);
    const float* from = a.partial;
    const int di = (int)d;
    if (param_dtype == VRS_F32)
      st = launch_after(qk_norm_rope_finish_kernel<float>, grid, 256, 0, s, from, blocks, di, (float*)dq_weight, (float*)dk_weight);
    else if (param_dtype == VRS_F16)
      st = launch_after(qk_norm_rope_finish_kernel<f16>, grid, 256, 0, s, from, blocks, di, (f16*)dq_weight, (f16*)dk_weight);
    else
      st = launch_after(qk_norm_rope_finish_kernel<bf16>, grid, 256, 0, s, from, blocks, di, (bf16*)dq_weight, (bf16*)dk_weight);
    if (st == VRS_OK) count_launch();
  }
  prof_end(t, s);
  return st;
}
