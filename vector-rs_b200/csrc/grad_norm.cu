// grad_norm.cu -- the norm over a list of gradients, and the gradients times
// the factor that brings it below a limit:
//   norm = unscale * sqrt(sum g^2),  out = g * unscale * min(1, max_norm / (norm + 1e-6)).
//
// Bound by memory: every gradient is read for the norm and, since the factor
// needs all of them, once more for the result. The list travels as kernel
// parameters, so a call copies nothing to the device and can be captured. Each
// tensor is cut into chunks of 16 KB, a block takes a run of neighbouring
// chunks: forward for the norm, backward for the result, which then finds in L2
// what the norm read last. In place and with a factor of 1 there is nothing to
// write, and the second pass ends at once.
//
// Squares are added in 32 bits within the 16 bytes of one load and in 64 bits
// beyond that: a 64-bit addition and conversion for 4 to 8 elements are far from
// bounding the pass. A group whose 32-bit sum may have overflowed or lost digits
// (f32 and bf16 reach 2^127 and 2^-126; their squares do not) is added again in
// 64 bits. Partial sums have one place a block and are added in order.
// 217 M elements of f16 into f32: norm 67 us (6.46 TB/s), result 224.
#include <cmath>
#include <type_traits>

#include "ops_common.cuh"

namespace vrs {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kLoads = 4;                          // 16-byte accesses of a thread in a chunk
constexpr int kChunkVecs = kThreads * kLoads;      // 16 KB
// Blocks a launch has at most: 8 of 256 threads on each of 148 SMs (a constant,
// so that the workspace does not depend on the device).
constexpr int kMostBlocks = 1184;
// Tensors a launch: its parameters take at most 32,764 bytes.
constexpr int kMostTensors = 1000;

struct Grad {
  const void* in;
  void* out;
  int64_t n;
  uint32_t chunk;   // the tensor's first chunk in the launch
  uint8_t type;     // of the gradient
  uint8_t out_f32;  // the result's type: 32 bits, or as the gradient
  uint8_t head;     // elements before the first 16-byte boundary
  uint8_t wide;     // results can be stored by whole accesses
};

struct Common {
  int tensors;
  uint32_t chunks;
  double* partial;
  int partials;    // of all launches
  int first;       // this launch's place among them
  float unscale, max_norm;
  float* norm;
  int write_norm;
  int in_place;    // all of them
};

template <int N>
struct Args : Common {
  Grad g[N];
};

template <class A>
__device__ __forceinline__ int tensor_of(const A& a, uint32_t chunk) {
  int lo = 0, hi = a.tensors;  // g[lo].chunk <= chunk < g[hi].chunk
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.g[mid].chunk <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <class T>
__device__ __forceinline__ void square_one(T v, double& acc) {
  const double d = (double)to_f32(v);
  acc = fma(d, d, acc);
}

// The squares of one access. (A 16-bit float's squares, 2^-48 to 2^32, keep
// their digits in 32 bits. The limits: sums below 2^-90 may hold squares below
// 2^-126, which have lost digits of theirs.)
template <class T, int VEC>
__device__ __forceinline__ void square_pack(const Pack<T, VEC>& p, double& acc) {
  F2 s = pack_f2(0.0f);
#pragma unroll
  for (int j = 0; j < VEC; j += 2) {
    const F2 v = pair_of(&p.v[j]);
    s = fma2(v, v, s);
  }
  const float sum = sum_f2(s);
  if (std::is_same<T, f16>::value) {
    acc += (double)sum;
    return;
  }
  if (sum > 0x1p-90f && sum < 0x1p126f) {
    acc += (double)sum;
    return;
  }
  const uint4 u = *reinterpret_cast<const uint4*>(&p);
  if (((u.x | u.y | u.z | u.w) & 0x7fff7fffu) == 0 && (sizeof(T) == 2 || ((u.x | u.y | u.z | u.w) & 0x7fffffffu) == 0))
    return;  // zeros
#pragma unroll
  for (int j = 0; j < VEC; j++) square_one(p.v[j], acc);
}

// A chunk of a tensor: whole accesses [0, vecs) from `at` on, and single
// elements before (the tensor's first chunk) and after them (its last).
struct Part {
  int64_t at;
  int vecs, before, after;
};
template <int VEC>
__device__ __forceinline__ Part part_of(const Grad& g, uint32_t chunk) {
  Part p;
  const int64_t c = (int64_t)(chunk - g.chunk) * kChunkVecs;
  const int head = (int)min((int64_t)g.head, g.n);
  const int64_t all = (g.n - head) / VEC;
  p.at = head + c * VEC;
  p.vecs = (int)max((int64_t)0, min((int64_t)kChunkVecs, all - c));
  p.before = c == 0 ? head : 0;
  p.after = c + kChunkVecs >= all ? (int)(g.n - head - all * VEC) : 0;
  return p;
}

template <class T>
__device__ __forceinline__ void norm_chunk(const Grad& g, uint32_t chunk, double& acc) {
  constexpr int VEC = 16 / sizeof(T);
  const Part p = part_of<VEC>(g, chunk);
  const T* in = (const T*)g.in;
  const T* at = in + p.at;
  const int tid = threadIdx.x;
  if (p.vecs == kChunkVecs) {
    Pack<T, VEC> v[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) v[i] = load_pack<T, VEC>(at + (i * kThreads + tid) * VEC);
#pragma unroll
    for (int i = 0; i < kLoads; i++) square_pack<T, VEC>(v[i], acc);
  } else {
    for (int i = tid; i < p.vecs; i += kThreads) square_pack<T, VEC>(load_pack<T, VEC>(at + i * VEC), acc);
  }
  if (tid < p.before) square_one(in[tid], acc);
  if (tid < p.after) square_one(at[p.vecs * VEC + tid], acc);
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s[kThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; w++) v += s[w];
  return v;
}

// Neighbouring chunks for each block, the first ones one more.
__device__ __forceinline__ void run_of(uint32_t chunks, uint32_t& c0, uint32_t& c1) {
  const uint32_t per = chunks / gridDim.x, more = chunks % gridDim.x, b = blockIdx.x;
  c0 = b * per + min(b, more);
  c1 = c0 + per + (b < more);
}

template <int N>
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ Args<N> a) {
  grid_launch();
  grid_wait();
  uint32_t c0, c1;
  run_of(a.chunks, c0, c1);
  double acc = 0.0;
  int t = c0 < c1 ? tensor_of(a, c0) : 0;
  for (uint32_t c = c0; c < c1; c++) {
    while (t + 1 < a.tensors && a.g[t + 1].chunk <= c) t++;
    const Grad g = a.g[t];
    if (g.type == VRS_F32)
      norm_chunk<float>(g, c, acc);
    else if (g.type == VRS_F16)
      norm_chunk<f16>(g, c, acc);
    else
      norm_chunk<bf16>(g, c, acc);
  }
  acc = block_sum(acc);
  if (threadIdx.x == 0) a.partial[a.first + blockIdx.x] = acc;
}

template <class T, class O>
__device__ __forceinline__ void store_one(O* o, T v, float f) {
  *o = from_f32<O>(to_f32(v) * f);
}

// Results are stored past the caches' reach (evict first): what is left of the
// gradients in L2 stays there for the chunks before.
template <class O, int VEC>
__device__ __forceinline__ void stream_pack(O* o, const float* v) {
  Pack<O, VEC> p;
#pragma unroll
  for (int j = 0; j < VEC; j += 2) round_pair(p.v + j, v[j], v[j + 1]);
  __stcs(reinterpret_cast<uint4*>(o), *reinterpret_cast<uint4*>(&p));
}

// Accesses of 16 bytes on the result's side: of 16-bit gradients that become 32-bit
// ones 8 bytes are read, so that neighbouring lanes store neighbouring 16 bytes.
template <class T, class O>
__device__ __forceinline__ void scale_chunk(const Grad& g, uint32_t chunk, float f) {
  constexpr int VEC = 16 / sizeof(T), W = 16 / sizeof(O), N = kLoads * VEC / W;
  const Part p = part_of<VEC>(g, chunk);
  const T* in = (const T*)g.in;
  O* out = (O*)g.out;
  const T* at = in + p.at;
  O* to = out + p.at;
  const int tid = threadIdx.x;
  auto put = [&](int i, const Pack<T, W>& k) {
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = to_f32(k.v[j]) * f;
    if (g.wide) {
      stream_pack<O, W>(to + i * W, v);
    } else {
#pragma unroll
      for (int j = 0; j < W; j++) to[i * W + j] = from_f32<O>(v[j]);
    }
  };
  if (p.vecs == kChunkVecs) {
    Pack<T, W> v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = load_pack<T, W>(at + (i * kThreads + tid) * W);
#pragma unroll
    for (int i = 0; i < N; i++) put(i * kThreads + tid, v[i]);
  } else {
    for (int i = tid; i < p.vecs * (VEC / W); i += kThreads) put(i, load_pack<T, W>(at + i * W));
  }
  if (tid < p.before) store_one(out + tid, in[tid], f);
  if (tid < p.after) store_one(to + p.vecs * VEC + tid, at[p.vecs * VEC + tid], f);
}

template <int N>
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ Args<N> a) {
  grid_launch();
  grid_wait();
  // Every block adds all partial sums, in one order.
  double acc = 0.0;
  for (int i = threadIdx.x; i < a.partials; i += kThreads) acc += a.partial[i];
  const double norm = sqrt(block_sum(acc)) * (double)a.unscale;
  if (a.write_norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
  if (a.tensors == 0) return;
  const double q = (double)a.max_norm / (norm + 1e-6);
  const float f = (float)((q >= 1.0 ? 1.0 : q) * (double)a.unscale);  // (a NaN stays one)
  if (f == 1.0f && a.in_place) return;
  uint32_t c0, c1;
  run_of(a.chunks, c0, c1);
  if (c0 >= c1) return;
  int t = tensor_of(a, c1 - 1);
  for (uint32_t c = c1; c-- > c0;) {
    while (a.g[t].chunk > c) t--;
    const Grad g = a.g[t];
    if (f == 1.0f && g.in == g.out) continue;
    if (g.type == VRS_F32)
      scale_chunk<float, float>(g, c, f);
    else if (g.type == VRS_F16)
      g.out_f32 ? scale_chunk<f16, float>(g, c, f) : scale_chunk<f16, f16>(g, c, f);
    else
      g.out_f32 ? scale_chunk<bf16, float>(g, c, f) : scale_chunk<bf16, bf16>(g, c, f);
  }
}

// One launch's tensors, in the smallest parameter block that holds them
// (parameters are copied with every launch).
template <int N>
int launch_one(const Common& c, const Grad* g, bool scale, cudaStream_t s) {
  Args<N> a;
  static_cast<Common&>(a) = c;
  for (int i = 0; i < c.tensors; i++) a.g[i] = g[i];
  const unsigned blocks = c.chunks < kMostBlocks ? (c.chunks ? c.chunks : 1) : kMostBlocks;
  VRS_TRY(launch_after(scale ? grad_scale_kernel<N> : grad_norm_kernel<N>, blocks, kThreads, 0, s, a));
  count_launch();
  return VRS_OK;
}

int launch(const Common& c, const Grad* g, bool scale, cudaStream_t s) {
  if (c.tensors <= 16) return launch_one<16>(c, g, scale, s);
  if (c.tensors <= 120) return launch_one<120>(c, g, scale, s);
  return launch_one<kMostTensors>(c, g, scale, s);
}

int64_t launches_of(int64_t tensors) { return tensors < 1 ? 1 : (tensors + kMostTensors - 1) / kMostTensors; }

int run(const char* who, const vrs_grad* grads, int64_t tensors, bool clip, float max_norm, float unscale, float* norm,
        void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  const std::string w(who);
  if (tensors < 0 || tensors > (1 << 24)) return invalid(w + ": tensors must be in 0..2^24");
  if (tensors && !grads) return invalid(w + ": null list");
  if (!norm) return invalid(w + ": null norm");
  if (!(unscale > 0.0f) || !(unscale < INFINITY)) return invalid(w + ": unscale must be positive and finite");
  if (clip && !(max_norm >= 0.0f)) return invalid(w + ": max_norm must be at least 0");
  if (!workspace || ((uintptr_t)workspace & 7)) return invalid(w + ": workspace must be 8-byte aligned");
  int64_t need = 0;
  VRS_TRY(vrs_grad_norm_workspace(tensors, &need));
  if (workspace_bytes < need) return invalid(w + ": workspace too small");
  int64_t left = 1ll << 42;  // keeps a launch's chunks below 2^31
  for (int64_t i = 0; i < tensors; i++) {
    const vrs_grad& g = grads[i];
    if (g.count < 0 || g.count > left) return invalid(w + ": counts must be at least 0 and 2^42 in all");
    left -= g.count;
    if (g.dtype < VRS_F32 || g.dtype > VRS_BF16) return invalid(w + ": dtype must be f32, f16 or bf16");
    const int bytes = dtype_bytes(g.dtype);
    if (g.count && !g.grad) return invalid(w + ": null gradient");
    if ((uintptr_t)g.grad % bytes) return invalid(w + ": a gradient off its type's alignment");
    if (!clip) continue;
    if (g.out_dtype != g.dtype && g.out_dtype != VRS_F32)
      return invalid(w + ": results are in the gradient's type or f32");
    if (g.count && !g.out) return invalid(w + ": null result");
    if ((uintptr_t)g.out % dtype_bytes(g.out_dtype)) return invalid(w + ": a result off its type's alignment");
    if (g.count && g.out == g.grad && g.out_dtype != g.dtype) return invalid(w + ": in place the type stays");
  }
  cudaStream_t s = (cudaStream_t)cuda_stream;
  ProfToken t = prof_begin(clip ? "clip_grad_norm" : "grad_norm", s);
  const int64_t launches = launches_of(tensors);
  Common c{};
  c.partial = (double*)workspace;
  c.unscale = unscale;
  c.max_norm = max_norm;
  c.norm = norm;
  int status = VRS_OK;
  int partials = 0;
  for (int pass = 0; pass < 2 && status == VRS_OK; pass++) {
    if (pass == 1 && !clip) {  // the norm alone: one block
      c.tensors = 0;
      c.chunks = 0;
      c.partials = partials;
      c.write_norm = 1;
      status = launch(c, nullptr, true, s);
      break;
    }
    int64_t at = 0;
    for (int64_t l = 0; l < launches && status == VRS_OK; l++) {
      Grad list[kMostTensors];
      uint32_t chunks = 0;
      int n = 0;
      c.in_place = 1;
      for (; at < tensors && n < kMostTensors; at++) {
        const vrs_grad& v = grads[at];
        if (v.count == 0) continue;
        const int bytes = dtype_bytes(v.dtype), ob = clip ? dtype_bytes(v.out_dtype) : bytes;
        const int64_t vec = 16 / bytes;
        Grad& g = list[n];
        g.in = v.grad;
        g.out = v.out;
        g.n = v.count;
        g.type = (uint8_t)v.dtype;
        g.out_f32 = clip && v.out_dtype == VRS_F32;
        if (v.out != v.grad) c.in_place = 0;
        g.head = (uint8_t)((16 - (uintptr_t)v.grad % 16) % 16 / bytes);
        g.wide = ((uintptr_t)v.out + (uintptr_t)g.head * ob) % 16 == 0;
        g.chunk = chunks;
        const int64_t vecs = v.count > g.head ? (v.count - g.head) / vec : 0;
        chunks += (uint32_t)(vecs ? (vecs + kChunkVecs - 1) / kChunkVecs : 1);
        n++;
      }
      c.tensors = n;
      c.chunks = chunks;
      c.first = pass == 0 ? partials : 0;
      c.partials = partials;
      c.write_norm = l == 0;
      if (pass == 0) partials += chunks < kMostBlocks ? (chunks ? (int)chunks : 1) : kMostBlocks;
      status = launch(c, list, pass == 1, s);
    }
  }
  prof_end(t, s);
  return status;
}

}  // namespace
}  // namespace ops
}  // namespace vrs

extern "C" int vrs_grad_norm_workspace(int64_t tensors, int64_t* out_bytes) {
  using namespace vrs::ops;
  if (tensors < 0 || tensors > (1 << 24) || !out_bytes)
    return invalid("vrs_grad_norm_workspace: tensors must be in 0..2^24 and out_bytes not null");
  *out_bytes = launches_of(tensors) * kMostBlocks * 8;
  return VRS_OK;
}

extern "C" int vrs_grad_norm(const vrs_grad* grads, int64_t tensors, float unscale, float* norm, void* workspace,
                             int64_t workspace_bytes, void* cuda_stream) {
  return vrs::ops::run("vrs_grad_norm", grads, tensors, false, 0.0f, unscale, norm, workspace, workspace_bytes,
                       cuda_stream);
}

extern "C" int vrs_clip_grad_norm(const vrs_grad* grads, int64_t tensors, float max_norm, float unscale, float* norm,
                                  void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  return vrs::ops::run("vrs_clip_grad_norm", grads, tensors, true, max_norm, unscale, norm, workspace, workspace_bytes,
                       cuda_stream);
}
