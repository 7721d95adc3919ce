// linear_ce.cu -- softmax cross entropy of scale * x table^T against one
// target a row, without keeping the scores, and its gradients:
//   z = scale x w_v, lse = log sum_v e^z, loss = lse - z[target]
//   g = (e^(z - lse) - [v = target]) dloss scale, dx = g table, dtable = g^T x.
// A row whose target lies outside the table takes no part: loss 0, lse 0, no
// gradient, whatever its values are. For v = target the bracket is e^-loss - 1,
// from the forward pass's loss: its difference to 1 would be lost in e^(z - lse).
//
// Forward it reads rows and table once (from memory; the products' tiles again
// from L2) and does 2 rows classes d operations, backward three times that:
// the scores are computed again rather than kept (rows x classes values would
// be read and written at some twice the products' time for d of some hundreds).
//
// This file holds the plan of a call and its small kernels; the products are
// in linear_ce_tc.cu.
//   forward   pack -> scores (maximum and sum per row and class tile) -> combine
//   backward  pack -> for each piece of the classes: gradient of the scores in
//             16 bits -> dx and dtable products -> finish
// `pack` copies the rows that take part next to one another (their count
// stays on the device and sets the number of tiles), so rows without a target
// cost nothing and their values, NaN too, reach no sum. It also gives the
// products an aligned operand whatever x's stride and address are.
#include <cmath>

#include <cudaTypedefs.h>

#include "linear_ce.cuh"

namespace vrs {
namespace ops {
namespace {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// Gradient of the scores held at a time.
constexpr int64_t kPieceBytes = 256ll << 20;
// CTA pairs that a product is split for (148 SMs). A constant, so that sums
// are split alike on every device.
constexpr int kPairs = 74;
// A product takes the score gradients as two 16-bit values each, the rounded one
// and the rest, and then adds nothing to the result's own rounding, where that
// rounding would show: in sums of up to kFewTerms terms (dtable: rows, dx:
// classes), and in problems of up to kTwoPlanes multiply-adds. One rounding of a
// lone term's gradient is common to a whole row of the result and at worst as
// large as the result's own half ulp; over n terms of one sign the roundings
// average to 1 / sqrt n of it, over terms of random signs they stay (in the
// root mean square) as large as the result's own, but differ between its elements.
// Few terms are one K block, so the second plane costs its writing and one K
// block more: backward 64 x 100,000 x 256 88 us with one, 95 with two; 20,000 x 17 x
// 130 64 and 69. Small problems show it in dx and dtable (8 x 1,398 x 75 in f16
// against 64 bits: up to 3.2e-4 with one, 2.0e-4 with two, as rounding the exact
// result leaves), larger ones would pay more: 128 x 8,192 x 256 25.9 and 32.0 us,
// 1,024 x 8,192 x 256 40 and 57.
constexpr int kFewTerms = kCeK;
constexpr int64_t kTwoPlanes = 1ll << 24;
// Up to here each pack block reads all targets itself; above, a first kernel
// counts them per kSlab rows.
constexpr int64_t kScanRows = 8192;
constexpr int kSlab = 1024;

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// ------------------------------------------------------------------- pack

struct Pack1 {
  const void* x;
  int64_t xs, rows;
  int d, dp;
  bool vec;  // 16-byte reads of x
  const int64_t* targets;
  int64_t classes;
  int per_block;
  int pack_blocks;  // the grid's other blocks copy the table
  const uint16_t* table;  // as given
  int64_t ts;
  uint16_t* table_out;
  const int2* slabs;  // per slab: taking rows, bits of the largest finite |dloss|; null: read all targets
  CeHeader* head;
  void* xc;        // [taking rows, tail zeros to a whole tile][dp]
  int* index;      // compact row -> row (forward)
  int* pos;        // row -> compact row or -1 (backward)
  int* target;
  // forward
  float* loss;
  float* lse_out;
  // backward
  const float* dloss;
  const float* lse;
  const float* losses;  // null: the target's scores are multiplied out again
  float scale;
  bool f16;
  float* lse2;
  float* gs;
  float* gy;
};

__device__ __forceinline__ bool takes_part(const Pack1& a, int64_t r) {
  const int64_t t = a.targets[r];
  return t >= 0 && t < a.classes;
}

// What a row's weight adds to the largest |dloss|: one that is not finite spoils
// its own row and must not scale the others'.
__device__ __forceinline__ unsigned weight_bits(float dloss) {
  const unsigned u = __float_as_uint(fabsf(dloss));
  return u < 0x7f800000u ? u : 0u;
}

// Sum, sum and maximum over a block of 256.
__device__ __forceinline__ void block_reduce(int& a, int& b, unsigned& m, int (*s)[3]) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(~0u, a, o);
    b += __shfl_xor_sync(~0u, b, o);
    m = max(m, __shfl_xor_sync(~0u, m, o));
  }
  if ((threadIdx.x & 31) == 0) {
    s[threadIdx.x >> 5][0] = a;
    s[threadIdx.x >> 5][1] = b;
    s[threadIdx.x >> 5][2] = (int)m;
  }
  __syncthreads();
  a = b = 0;
  m = 0;
#pragma unroll
  for (int w = 0; w < 8; w++) {
    a += s[w][0];
    b += s[w][1];
    m = max(m, (unsigned)s[w][2]);
  }
}

__global__ void __launch_bounds__(256) ce_count_kernel(const Pack1 a, int2* slabs) {
  __shared__ int s[8][3];
  int n = 0, none = 0;
  unsigned m = 0;
  const int64_t r0 = (int64_t)blockIdx.x * kSlab;
  for (int64_t r = r0 + threadIdx.x; r < min(a.rows, r0 + kSlab); r += 256)
    if (takes_part(a, r)) {
      n++;
      if (a.dloss) m = max(m, weight_bits(a.dloss[r]));
    }
  block_reduce(n, none, m, s);
  if (threadIdx.x == 0) slabs[blockIdx.x] = make_int2(n, (int)m);
}

// The score gradients are rounded to 16 bits relative to the largest
// finite |dloss|: with one weight for all rows (a mean) the target's -1 stays
// exact and no weight's own rounding biases the sums. Where it is 0: to 1.
__device__ __forceinline__ float grad_unit(unsigned max_bits) {
  const float m = __uint_as_float(max_bits);
  return m > 0.0f ? m : 1.0f;
}
// f16 ends at 2^16 and loses bits below 2^-14: its gradients use the range up to 2^13.
constexpr float kF16Gain = 8192.0f;

// One row of d elements at any address, copied by a warp to `to` (16-byte
// aligned, dp elements, zeros past d). Where whole 16-byte words around the row
// may be read (`inside`), each lane reads the two that its 16 bytes lie in and
// shifts them into place; else the row is read element by element.
__device__ __forceinline__ void copy_row(const uint16_t* from, int d, int dp, uint16_t* to, bool inside) {
  const int lane = threadIdx.x & 31, chunks = dp / 8;
  uint4* out = reinterpret_cast<uint4*>(to);
  if (!inside) {
    for (int c = lane; c < chunks; c += 32) {
      Pack<uint16_t, 8> q;
#pragma unroll
      for (int j = 0; j < 8; j++) q.v[j] = c * 8 + j < d ? from[c * 8 + j] : 0;
      out[c] = *reinterpret_cast<uint4*>(&q);
    }
    return;
  }
  const uint4* in = reinterpret_cast<const uint4*>((uintptr_t)from & ~(uintptr_t)15);
  const int shift = (int)((uintptr_t)from & 15);  // bytes, even; the same for the warp
  constexpr int U = 4;
  for (int c0 = lane; c0 < chunks; c0 += 32 * U) {
    uint4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = c0 + 32 * u;
      if (c < chunks) {
        lo[u] = in[c];
        hi[u] = make_uint4(0, 0, 0, 0);
        if (2 * (d - c * 8) > 16 - shift) hi[u] = in[c + 1];  // else no element lies in it
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = c0 + 32 * u;
      if (c >= chunks) continue;
      uint32_t w[8] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w};
      if (shift & 8) {
#pragma unroll
        for (int j = 0; j < 6; j++) w[j] = w[j + 2];
      }
      if (shift & 4) {
#pragma unroll
        for (int j = 0; j < 5; j++) w[j] = w[j + 1];
      }
      if (shift & 2) {
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
      }
      const int left = d - c * 8;
      if (left < 8) {
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = left >= 2 * j + 2 ? w[j] : left == 2 * j + 1 ? w[j] & 0xffffu : 0u;
      }
      out[c] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <bool BACK>
__global__ void __launch_bounds__(256) ce_pack_kernel(const Pack1 a) {
  grid_launch();
  grid_wait();
  if ((int)blockIdx.x >= a.pack_blocks) {
    // The table's rows, a warp each. The 16-byte words around a row belong to
    // the table but for its first and last rows (and rows shorter than a word).
    const int64_t step = (int64_t)(gridDim.x - a.pack_blocks) * 8;
    for (int64_t v = (int64_t)(blockIdx.x - a.pack_blocks) * 8 + (threadIdx.x >> 5); v < a.classes; v += step)
      copy_row(a.table + v * a.ts, a.d, a.dp, a.table_out + v * a.dp, v > 0 && v < a.classes - 1 && a.d >= 8);
    return;
  }
  __shared__ int s[8][3];
  __shared__ int s_warp[8];
  __shared__ int s_row[256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * a.per_block;
  const int64_t r1 = min(a.rows, r0 + a.per_block);
  // Taking rows before this block's, and in all.
  int before = 0, total = 0;
  unsigned top = 0;
  if (a.slabs) {
    const int64_t slab = r0 / kSlab, n = (a.rows + kSlab - 1) / kSlab;
    for (int64_t i = tid; i < n; i += 256) {
      const int2 c = a.slabs[i];
      total += c.x;
      if (i < slab) before += c.x;
      top = max(top, (unsigned)c.y);
    }
    for (int64_t r = slab * kSlab + tid; r < r0; r += 256) before += takes_part(a, r);
  } else {
    // (Both loads of a row at once, sixteen rows in flight.)
#pragma unroll 16
    for (int64_t r = tid; r < a.rows; r += 256) {
      const int64_t t = a.targets[r];
      const unsigned g = BACK ? weight_bits(a.dloss[r]) : 0;
      if (t >= 0 && t < a.classes) {
        total++;
        before += r < r0;
        top = max(top, g);
      }
    }
  }
  block_reduce(before, total, top, s);
  const float unit = BACK ? grad_unit(top) : 1.0f, gain = BACK && a.f16 ? kF16Gain : 1.0f;
  if (blockIdx.x == 0 && tid == 0) {
    a.head->taken = total;
    a.head->grad_scale = unit * a.scale / gain;
  }
  // Places of this block's rows, in row order.
  const int64_t r = r0 + tid;
  const bool mine = r < r1, in = mine && takes_part(a, r);
  const unsigned bal = __ballot_sync(~0u, in);
  if (lane == 0) s_warp[warp] = __popc(bal);
  __syncthreads();
  int here = 0, n_in = 0;
#pragma unroll
  for (int w = 0; w < 8; w++) {
    here += w < warp ? s_warp[w] : 0;
    n_in += s_warp[w];
  }
  here += __popc(bal & ((1u << lane) - 1));
  if (in) {
    s_row[here] = tid;
    const int p = before + here;
    a.target[p] = (int)a.targets[r];
    if (BACK) {
      a.lse2[p] = a.lse[r] * kLog2e;
      a.gs[p] = a.dloss[r] / unit * gain;
      if (a.losses) a.gy[p] = expm1f(-a.losses[r]);
    } else {
      a.index[p] = (int)r;
    }
  }
  if (mine) {
    if (BACK) {
      a.pos[r] = in ? before + here : -1;
    } else if (!in) {
      a.loss[r] = 0.0f;
      a.lse_out[r] = 0.0f;
    }
  }
  __syncthreads();
  // One warp a row; elements past d are zeros.
  uint16_t* xc = (uint16_t*)a.xc;
  const uint16_t* x = (const uint16_t*)a.x;
  const int chunks = a.dp / 8;
  for (int i = warp; i < n_in; i += 8) {
    const int64_t row = r0 + s_row[i];
    uint16_t* to = xc + (int64_t)(before + i) * a.dp;
    if (a.vec) {
      const uint4* from = reinterpret_cast<const uint4*>(x + row * a.xs);
#pragma unroll 4
      for (int c = lane; c < chunks; c += 32) reinterpret_cast<uint4*>(to)[c] = from[c];
    } else {
      copy_row(x + row * a.xs, a.d, a.dp, to, row > 0 && row < a.rows - 1 && a.d >= 8);
    }
    if (BACK && !a.losses) {
      const uint16_t *from = x + row * a.xs, *w = a.table + a.targets[row] * a.ts;
      const bool vec = (((uintptr_t)from | (uintptr_t)w) & 15) == 0;
      const float z = __fmul_rn(a.f16 ? dot_rows<true>(from, w, a.d, vec) : dot_rows<false>(from, w, a.d, vec), a.scale);
      if (lane == 0) a.gy[before + i] = expm1f(z - a.lse[row]);
    }
  }
  // (Past the last row TMA reads zeros itself.)
  const int64_t tail = min(a.rows, (int64_t)(total + kCeM - 1) / kCeM * kCeM);
  for (int64_t p = total + (int64_t)blockIdx.x * 8 + warp; p < tail; p += (int64_t)a.pack_blocks * 8) {
    uint4* to = reinterpret_cast<uint4*>(xc + p * a.dp);
    for (int c = lane; c < chunks; c += 32) to[c] = make_uint4(0, 0, 0, 0);
  }
}

// --------------------------------------------------------- combine, finish

// (maximum, sum of powers of two below it) of two sets.
__device__ __forceinline__ float2 merge(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), sub = m == -INFINITY ? 0.0f : m;
  return make_float2(m, a.y * ex2(a.x - sub) + b.y * ex2(b.x - sub));
}

// loss and lse of rows from their parts' maxima and sums (in units of log 2) and
// the target's score z: with r the sum of the others' powers relative to the
// target's, loss = log(1 + r) where the target is the largest, and then lse = z +
// loss. (lse - z would leave a loss that is small against z the last bits of lse
// only: 1e-2 of a loss of 1e-4 at a score of 18.) Else the differences to z are
// taken before the logarithm's sum is rounded. z is rounded by itself, not within
// a sum, so that the backward pass can form the same lse - z. A block takes R
// rows (a power of two up to 32), 1024 / R threads each; the parts lie row by row.
// One warp a row multiplies the target's score out while the others' loads are
// on their way.
template <bool F16>
__global__ void __launch_bounds__(1024)
    ce_combine_kernel(const CeGemm a, int R, const int* __restrict__ index, float* loss, float* lse) {
  __shared__ float2 s[1024];
  grid_wait();
  const int taken = a.rows >= 0 ? a.rows : a.head->taken;
  const int64_t r0 = (int64_t)blockIdx.x * R;
  if (r0 >= taken) return;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool mine = w < R && r0 + w < taken;  // this warp's row
  int64_t tgt = -1;
  float z = 0.0f;
  if (mine) {
    tgt = index ? a.target[r0 + w] : a.targets[r0 + w];
    if (tgt >= 0 && tgt < a.classes)
      z = __fmul_rn(dot_rows<F16>(a.x + (r0 + w) * a.xs, a.w + tgt * a.ws, a.d, true), a.scale);
    else
      tgt = -1;
  }
  const int64_t row = r0 + threadIdx.x % R;
  const int strips = 1024 / R;
  float2 v = make_float2(-INFINITY, 0.0f);
  if (row < taken) {
    const float2* p = a.part + row;
#pragma unroll 8
    for (int i = threadIdx.x / R; i < a.parts; i += strips) v = merge(v, p[i * a.part_rows]);
  }
  s[threadIdx.x] = v;
  __syncthreads();
  if (!mine) return;
  v = make_float2(-INFINITY, 0.0f);
  for (int k = lane; k < strips; k += 32) v = merge(v, s[k * R + w]);
#pragma unroll
  for (int o = 16; o; o >>= 1) v = merge(v, make_float2(__shfl_xor_sync(~0u, v.x, o), __shfl_xor_sync(~0u, v.y, o)));
  if (lane == 0) {
    const int64_t at = index ? index[r0 + w] : r0 + w;
    float all = 0.0f, less = 0.0f;
    if (tgt >= 0) {
      const float z2 = z * kLog2e;
      if (v.x <= z2) {
        less = log1pf(v.y * exp2f(v.x - z2));
        all = z + less;
        if (isinf(z)) less = all - z;  // no loss: NaN
      } else {
        all = (v.x + log2f(v.y + exp2f(z2 - v.x))) * kLn2;
        less = ((v.x - z2) + log2f(v.y + exp2f(z2 - v.x))) * kLn2;
      }
    }
    lse[at] = all;
    loss[at] = less;
  }
}

// out[row] = sum over splits of acc[split][pos[row]], rounded once; rows
// without a place get zeros. A warp takes 128 columns of a row at a time.
template <class T>
__global__ void __launch_bounds__(256)
    ce_finish_kernel(const float* __restrict__ acc, int splits, int64_t split_rows, int d, int d4, int64_t rows,
                     const int* __restrict__ pos, const CeHeader* head, T* out, int64_t os, bool vec) {
  grid_wait();
  const float f = head->grad_scale;
  const int chunks = (d4 + 127) / 128;
  const int64_t step = (int64_t)gridDim.x * 8, units = rows * chunks;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
    const int64_t r = units < (1ll << 31) ? (int64_t)((uint32_t)u / (uint32_t)chunks) : u / chunks;
    const int c = (int)(u - r * chunks) * 128 + (threadIdx.x & 31) * 4;
    if (c >= d4) continue;
    const int64_t p = pos ? pos[r] : r;
    T* o = out + r * os + c;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (p >= 0) {
#pragma unroll 8
      for (int k = 0; k < splits; k++) {
        const float4 q = *reinterpret_cast<const float4*>(acc + (k * split_rows + p) * d4 + c);
        v.x += q.x;
        v.y += q.y;
        v.z += q.z;
        v.w += q.w;
      }
    }
    const float e[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
    if (vec) {
      store_pack<T, 4>(o, e);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (c + j < d) o[j] = from_f32<T>(e[j]);
    }
  }
}

template <class T>
int launch_finish(const float* acc, int splits, int64_t split_rows, int d, int d4, int64_t rows, const int* pos,
                  const CeHeader* head, void* out, int64_t os, cudaStream_t s) {
  const bool vec = d % 4 == 0 && (rows == 1 || os % 4 == 0) && (uintptr_t)out % 8 == 0;
  int sms = 0;
  VRS_TRY(sm_count(&sms));
  const int64_t need = (rows * ((d4 + 127) / 128) + 7) / 8, most = (int64_t)sms * 8;
  VRS_TRY(launch_after(ce_finish_kernel<T>, (unsigned)(need < most ? need : most), 256, 0, s, acc, splits, split_rows, d,
                       d4, rows, pos, head, (T*)out, os, vec));
  count_launch();
  return VRS_OK;
}

// ------------------------------------------------------------- host plan

// Offsets into the workspace, and how the work is cut. Nothing here depends on
// addresses or on which gradients are asked for, so neither do the sums. The room
// for what depends on the cut is a bound that never falls as a size grows, so that
// a workspace for the largest sizes serves all smaller ones.
struct Plan {
  int64_t rows_p, dp, d4;         // rows in whole tiles, row pitches
  int64_t piece;                  // classes of a piece, whole tiles
  int64_t vtiles;                 // class tiles in all
  int64_t parts;                  // and parts of 128 classes
  int splits_dx, splits_dw;
  int planes, planes_dx, planes_dw;  // of the score gradients: written, and taken by each product
  int64_t head, slabs, index, pos, target, lse2, gs, gy, xc, wc, part, g, acc_dx, acc_dw, bytes;
};

// Class tiles of a piece: few pieces of one size, as many (up to twice the
// fewest) as make the pairs' last turns fullest. A turn's length is that of its
// longest tile; the products' tiles are counted as the kernel orders them.
int64_t piece_of(int64_t rows_p, int planes, int64_t vtiles, int64_t ntiles) {
  int64_t most = kPieceBytes / (planes * rows_p * 2) / kCeN;
  most = most < 1 ? 1 : most < vtiles ? most : vtiles;
  const int64_t fewest = (vtiles + most - 1) / most, mt = rows_p / kCeM;
  int64_t best = most;
  double best_cost = 0.0;
  for (int64_t n = fewest; n <= 2 * fewest && n <= vtiles && n < fewest + 16; n++) {
    const int64_t vt = (vtiles + n - 1) / n;
    const double grad = (double)((mt * vt + kPairs - 1) / kPairs);
    // dx: mt * ntiles tiles of vt * 4 K blocks; dtable: vt * ntiles of mt * 4.
    const double l = (double)(mt > vt ? mt : vt), s = (double)(mt > vt ? vt : mt);
    const int64_t nl = (mt > vt ? vt : mt) * ntiles, ns = (mt > vt ? mt : vt) * ntiles;
    const int64_t turns = nl / kPairs, rem = nl % kPairs;
    const double left = (double)ns - (rem ? (double)(kPairs - rem) * std::floor(l / s + 0.5) : 0.0);
    const double store = (double)(turns + (rem != 0)) * l + (left > 0 ? std::ceil(left / kPairs) * s : 0.0);
    const double cost = (double)n * (grad * (double)ntiles + store + 2.0);
    if (best_cost == 0.0 || cost < best_cost) {
      best_cost = cost;
      best = vt;
    }
  }
  return best;
}

Plan make_plan(int64_t rows, int64_t classes, int64_t d, bool back, bool aligned) {
  Plan p{};
  p.rows_p = up(rows, kCeM);
  p.dp = up(d, 8);
  p.d4 = up(d, 4);
  p.vtiles = (classes + kCeN - 1) / kCeN;
  p.parts = (classes + 127) / 128;
  int64_t at = 0;
  // The smaller of what all of it takes and a limit, but room for one piece at least.
  auto most = [](int64_t all, int64_t limit, int64_t least) {
    const int64_t b = all < limit ? all : limit;
    return b > least ? b : least;
  };
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  p.head = take(sizeof(CeHeader));
  p.slabs = take(rows > kScanRows ? (rows + kSlab - 1) / kSlab * (int64_t)sizeof(int2) : 0);
  p.target = take(rows * 4);
  p.xc = take(p.rows_p * p.dp * 2);
  p.wc = take(aligned ? 0 : classes * p.dp * 2);
  if (!back) {
    p.index = take(rows * 4);
    p.part = take(rows * p.parts * (int64_t)sizeof(float2));
  } else {
    p.pos = take(rows * 4);
    p.lse2 = take(rows * 4);
    p.gs = take(rows * 4);
    p.gy = take(rows * 4);
    const bool small = rows * classes <= kTwoPlanes / d;
    p.planes_dx = small || classes <= kFewTerms ? 2 : 1;
    p.planes_dw = small || rows <= kFewTerms ? 2 : 1;
    p.planes = p.planes_dx > p.planes_dw ? p.planes_dx : p.planes_dw;
    p.piece = piece_of(p.rows_p, p.planes, p.vtiles, (d + kCeN - 1) / kCeN) * kCeN;
    // Room for two planes whether a problem has them or not.
    p.g = take(most(2 * p.rows_p * 2 * kCeN * p.vtiles, kPieceBytes, 2 * p.rows_p * 2 * kCeN));
    // Few tiles: K is split until the pairs have one each, 8 blocks deep at least.
    auto splits = [](int64_t tiles_, int64_t kblocks) {
      int64_t s = kPairs / tiles_ < kblocks / 8 ? kPairs / tiles_ : kblocks / 8;
      return (int)(s < 1 ? 1 : s);
    };
    const int64_t nt = (d + kCeN - 1) / kCeN;
    p.splits_dx = splits(p.rows_p / kCeM * nt, p.planes_dx * (p.piece / kCeK));
    p.splits_dw = splits(p.piece / kCeM * nt, p.planes_dw * ((rows + kCeK - 1) / kCeK));
    // A split product's tiles are at most kPairs, and its splits one per eight K blocks.
    const int64_t row_bytes = p.d4 * 4, tiles_bytes = kPairs * (int64_t)kCeM * kCeN * 4;
    const int64_t most_dx = 2 * (p.vtiles * kCeN / kCeK) / 8, most_dw = 2 * ((rows + kCeK - 1) / kCeK) / 8;
    const int64_t one = p.rows_p * row_bytes;
    p.acc_dx = take(most((most_dx < kPairs ? most_dx : kPairs) * one, tiles_bytes, one));
    p.acc_dw = take(most_dw < 2 ? 0
                                : most((most_dw < kPairs ? most_dw : kPairs) * p.vtiles * kCeN * row_bytes, tiles_bytes, 0));
  }
  p.bytes = at;
  return p;
}

int check(const std::string& who, int64_t rows, int64_t classes, int64_t d, int32_t dtype) {
  if (dtype != VRS_F16 && dtype != VRS_BF16)
    return invalid(who + ": rows and table are f16 or bf16 (operands of the tensor cores)");
  if (rows < 0 || rows > (1ll << 31) - 512) return invalid(who + ": rows must be in 0..2^31-512");
  if (classes < 1 || classes > (1ll << 31) - 512) return invalid(who + ": classes must be in 1..2^31-512");
  if (d < 1 || d > 65536) return invalid(who + ": d must be in 1..65536");
  if (rows > (1ll << 46) / classes) return invalid(who + ": rows x classes must be at most 2^46");
  return VRS_OK;
}

int check_scale(const std::string& who, float scale) {
  if (!(scale > 0.0f) || !std::isfinite(scale)) return invalid(who + ": scale must be positive and finite");
  return VRS_OK;
}

int check_workspace(const std::string& who, const void* ws, int64_t have, int64_t need) {
  if (!ws) return invalid(who + ": null workspace");
  if ((uintptr_t)ws % 256) return invalid(who + ": workspace must be 256-byte aligned");
  if (have < need)
    return invalid(who + ": workspace of " + std::to_string(have) + " bytes, " + std::to_string(need) + " needed");
  return VRS_OK;
}

// Rows that TMA can address: 16-byte aligned starts.
bool tma_rows(const void* p, int64_t stride, int64_t rows) { return aligned16(p) && (rows == 1 || stride % 8 == 0); }

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// [rows][inner] row-major with `stride` elements between rows; boxes of 128
// bytes by box_rows, 128-byte swizzle, zeros outside.
int make_map(CUtensorMap* m, CUtensorMapDataType type, int bytes, const void* base, int64_t inner, int64_t rows,
             int64_t stride, int box_rows) {
  auto fn = encode_fn();
  if (!fn) {
    set_error(VRS_ERR_DRIVER, "cuTensorMapEncodeTiled unavailable");
    return VRS_ERR_DRIVER;
  }
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(rows == 1 ? up(inner * bytes, 16) : stride * bytes)};
  cuuint32_t box[2] = {(cuuint32_t)(128 / bytes), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(VRS_ERR_DRIVER, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
    return VRS_ERR_DRIVER;
  }
  return VRS_OK;
}

struct Call {
  const void* x;
  int64_t xs, rows;
  const void* table;
  int64_t ts, classes, d;
  int32_t dtype;
  const int64_t* targets;
  float scale;
  char* ws;
  cudaStream_t s;
};

// Packs the rows (and the table where TMA cannot address it) and fills what
// both passes' products share. Forward, up to one tile of rows that TMA can
// address stay where they are: there are no tiles to save, and a row's values
// reach its own loss only.
int start(const Call& c, const Plan& p, Pack1& k, CeMaps& maps, CeGemm& a, bool back) {
  int* err = nullptr;
  VRS_TRY(error_word(&err));
  int sms = 0;
  VRS_TRY(sm_count(&sms));
  k.x = c.x;
  k.xs = c.rows == 1 ? 0 : c.xs;
  k.rows = c.rows;
  k.d = (int)c.d;
  k.dp = (int)p.dp;
  k.vec = c.d % 8 == 0 && tma_rows(c.x, c.xs, c.rows);
  k.targets = c.targets;
  k.classes = c.classes;
  k.head = (CeHeader*)(c.ws + p.head);
  k.xc = c.ws + p.xc;
  k.target = (int*)(c.ws + p.target);
  const void* w = c.table;
  int64_t ts = c.ts;
  const bool copied = !tma_rows(w, ts, c.classes);
  const bool packed = back || copied || c.rows > kCeM || !tma_rows(c.x, c.xs, c.rows);
  a.rows = packed ? -1 : (int)c.rows;
  if (packed) {
    if (c.rows > kScanRows) {
      int2* slabs = (int2*)(c.ws + p.slabs);
      ce_count_kernel<<<(unsigned)((c.rows + kSlab - 1) / kSlab), 256, 0, c.s>>>(k, slabs);
      VRS_CUDA(cudaGetLastError());
      count_launch();
      k.slabs = slabs;
      k.per_block = 64;
    } else {
      k.per_block = (int)((c.rows + 2 * sms - 1) / (2 * sms));
    }
    k.pack_blocks = (int)((c.rows + k.per_block - 1) / k.per_block);
    int64_t blocks = k.pack_blocks;
    k.table = (const uint16_t*)w;
    k.ts = c.classes == 1 ? 0 : ts;
    if (copied) {
      k.table_out = (uint16_t*)(c.ws + p.wc);
      const int64_t need = (c.classes + 7) / 8, most = (int64_t)sms * 16;
      blocks += need < most ? need : most;
      w = k.table_out;
      ts = p.dp;
    }
    VRS_TRY(launch_after(back ? ce_pack_kernel<true> : ce_pack_kernel<false>, (unsigned)blocks, 256, 0, c.s, k));
    count_launch();
  } else {
    a.targets = c.targets;
  }
  const bool f16 = c.dtype == VRS_F16;
  const CUtensorMapDataType type = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // K-major loads of the rows take 128 of them (64 where there are no more),
  // those of the table 64.
  a.one_tile_rows = c.rows <= kCeM ? (int)c.rows : 0;
  const int box = a.one_tile_rows && c.rows <= 64 ? 64 : 128;
  VRS_TRY(make_map(&maps.a0, type, 2, packed ? k.xc : c.x, c.d, c.rows, packed ? p.dp : c.xs, box));
  VRS_TRY(make_map(&maps.b0, type, 2, w, c.d, c.classes, ts, 64));
  a.x = (const uint16_t*)(packed ? k.xc : c.x);
  a.xs = packed ? p.dp : c.rows == 1 ? 0 : c.xs;
  a.w = (const uint16_t*)w;
  a.ws = c.classes == 1 ? 0 : ts;
  a.head = k.head;
  a.err = err;
  a.classes = (int)c.classes;
  a.d = (int)c.d;
  a.kblocks = (int)((c.d + kCeK - 1) / kCeK);
  // kind::f16, f32 accumulator; operand types by bits 7 and 10.
  a.idesc = (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10));
  a.target = k.target;
  a.scale = c.scale;
  a.c2 = c.scale * kLog2e;
  return VRS_OK;
}

int forward(const Call& c, const Plan& p, float* loss, float* lse) {
  Pack1 k{};
  CeMaps maps;
  CeGemm a{};
  k.index = (int*)(c.ws + p.index);
  k.loss = loss;
  k.lse_out = lse;
  VRS_TRY(start(c, p, k, maps, a, false));
  a.vn = a.classes;
  // One tile of rows reads the table at the speed of memory: where at most
  // half of the CTAs or pairs would have a tile in the last turn, halves of
  // tiles shorten it.
  const int64_t units = ce_single(a.one_tile_rows) ? 2 * kPairs : kPairs, rest = p.vtiles % units;
  a.whole = (int)(c.rows <= kCeM && 2 * rest <= units ? p.vtiles - rest : p.vtiles);
  a.vtiles = a.whole == p.vtiles ? a.whole : a.whole + (int)((c.classes - a.whole * (int64_t)kCeN + 127) / 128);
  a.parts = (int)p.parts;
  a.part_rows = c.rows;
  a.part = (float2*)(c.ws + p.part);
  VRS_TRY(launch_ce_gemm(kCeLse, c.dtype == VRS_F16, maps, a, p.rows_p / kCeM * a.vtiles, c.s));
  const int* index = a.rows < 0 ? k.index : nullptr;
  // Up to 32 rows a block (whole lines of parts), fewer where blocks are few.
  int R = 1;
  while (R < 32 && R < c.rows && (R < 4 || c.rows > R * 256)) R *= 2;
  VRS_TRY(launch_after(c.dtype == VRS_F16 ? ce_combine_kernel<true> : ce_combine_kernel<false>,
                       (unsigned)((c.rows + R - 1) / R), 1024, 0, c.s, a, R, index, loss, lse));
  count_launch();
  return VRS_OK;
}

int finish(bool f16, const float* acc, int splits, int64_t split_rows, const Plan& p, int64_t d, int64_t rows,
           const int* pos, const CeHeader* head, void* out, int64_t os, cudaStream_t s) {
  return f16 ? launch_finish<ops::f16>(acc, splits, split_rows, (int)d, (int)p.d4, rows, pos, head, out, os, s)
             : launch_finish<bf16>(acc, splits, split_rows, (int)d, (int)p.d4, rows, pos, head, out, os, s);
}

int backward(const Call& c, const Plan& p, const float* dloss, const float* lse, const float* losses, void* dx,
             int64_t dxs, void* dtable, int64_t dts) {
  const bool f16 = c.dtype == VRS_F16;
  const CUtensorMapDataType type = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  Pack1 k{};
  CeMaps maps;
  CeGemm a{};
  k.pos = (int*)(c.ws + p.pos);
  k.dloss = dloss;
  k.lse = lse;
  k.losses = losses;
  k.scale = c.scale;
  k.f16 = f16;
  k.lse2 = (float*)(c.ws + p.lse2);
  k.gs = (float*)(c.ws + p.gs);
  k.gy = (float*)(c.ws + p.gy);
  VRS_TRY(start(c, p, k, maps, a, true));
  a.lse2 = k.lse2;
  a.gs = k.gs;
  a.gy = k.gy;
  float* acc_dx = (float*)(c.ws + p.acc_dx);
  float* acc_dw = (float*)(c.ws + p.acc_dw);
  VRS_TRY(make_map(&maps.out0, type, 2, c.ws + p.g, p.piece, p.rows_p, p.piece, 32));
  CeMaps prod;  // of the products
  VRS_TRY(make_map(&prod.a0, type, 2, c.ws + p.g, p.piece, p.planes * p.rows_p, p.piece, 128));
  VRS_TRY(make_map(&prod.a1, type, 2, c.ws + p.g, p.piece, p.planes * p.rows_p, p.piece, 64));
  a.planes = p.planes;
  a.plane_rows = (int)p.rows_p;
  a.g = (uint16_t*)(c.ws + p.g);
  a.g_pitch = p.piece;
  VRS_TRY(make_map(&prod.b1, type, 2, k.xc, c.d, c.rows, p.dp, 64));
  prod.b0 = maps.b0;
  a.dx.on = dx != nullptr;
  a.dw.on = dtable != nullptr;
  a.dx.ntiles = a.dw.ntiles = (int)((c.d + kCeN - 1) / kCeN);
  a.dx.splits = p.splits_dx;
  a.dw.splits = p.splits_dw;
  a.dx.planes = p.planes_dx;
  a.dw.planes = p.planes_dw;
  a.d4 = (int)p.d4;
  a.dx.f32 = acc_dx;
  a.dx.f32_rows = (int)p.rows_p;
  const bool direct = p.splits_dw == 1;
  if (dtable) {
    if (!direct) {
      a.dw.f32 = acc_dw;
      a.dw.f32_rows = (int)p.piece;
    } else {
      a.dw.out = (uint16_t*)dtable;
      a.dw.out_stride = c.classes == 1 ? 0 : dts;
      a.dw.out_vec = c.d % 8 == 0 && tma_rows(dtable, dts, c.classes);
    }
  }
  for (int64_t v0 = 0; v0 < c.classes; v0 += p.piece) {
    const int64_t vn = c.classes - v0 < p.piece ? c.classes - v0 : p.piece;
    a.v0 = (int)v0;
    a.vn = (int)vn;
    a.vtiles = a.whole = (int)((vn + kCeN - 1) / kCeN);
    VRS_TRY(launch_ce_gemm(kCeGrad, f16, maps, a, p.rows_p / kCeM * a.vtiles, c.s));
    a.dx.kblocks = (int)((vn + kCeK - 1) / kCeK);
    a.dx.add = v0 > 0;
    a.dw.mtiles = a.vtiles;
    a.dw.row0 = (int)v0;
    const int64_t tiles = (dx ? p.rows_p / kCeM * a.dx.ntiles * a.dx.splits : 0) +
                          (dtable ? (int64_t)a.dw.mtiles * a.dw.ntiles * a.dw.splits : 0);
    VRS_TRY(launch_ce_gemm(kCeStore, f16, prod, a, tiles, c.s));
    if (dtable && !direct)
      VRS_TRY(finish(f16, acc_dw, p.splits_dw, p.piece, p, c.d, vn, nullptr, a.head, (char*)dtable + v0 * dts * 2, dts,
                     c.s));
  }
  if (dx) VRS_TRY(finish(f16, acc_dx, p.splits_dx, p.rows_p, p, c.d, c.rows, k.pos, a.head, dx, dxs, c.s));
  return VRS_OK;
}

}  // namespace
}  // namespace ops
}  // namespace vrs

extern "C" int vrs_linear_cross_entropy_workspace(int64_t rows, int64_t classes, int64_t d, int32_t dtype,
                                                  int32_t backward, int32_t aligned, int64_t* out_bytes) {
  using namespace vrs::ops;
  const char* who = "vrs_linear_cross_entropy_workspace";
  if (!out_bytes) return invalid(std::string(who) + ": null out_bytes");
  VRS_TRY(check(who, rows, classes, d, dtype));
  *out_bytes = rows == 0 ? 0 : make_plan(rows, classes, d, backward != 0, aligned != 0).bytes;
  return VRS_OK;
}

extern "C" int vrs_linear_cross_entropy_forward(const void* x, int64_t x_stride, int64_t rows, const void* table,
                                                int64_t table_stride, int64_t classes, int64_t d, int32_t dtype,
                                                const int64_t* targets, float scale, float* loss, float* lse,
                                                void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  const std::string who = "vrs_linear_cross_entropy_forward";
  VRS_TRY(check(who, rows, classes, d, dtype));
  VRS_TRY(check_scale(who, scale));
  if (rows == 0) return VRS_OK;
  if (!x || !table || !targets || !loss || !lse) return invalid(who + ": null buffer");
  if ((rows > 1 && x_stride < d) || (classes > 1 && table_stride < d))
    return invalid(who + ": row strides must be at least d");
  const Plan p = make_plan(rows, classes, d, false, tma_rows(table, table_stride, classes));
  VRS_TRY(check_workspace(who, workspace, workspace_bytes, p.bytes));
  const Call c{x,       x_stride, rows,  table, table_stride, classes, d, dtype, targets, scale, (char*)workspace,
               (cudaStream_t)cuda_stream};
  ProfToken t = prof_begin("linear_cross_entropy_forward", c.s);
  const int st = forward(c, p, loss, lse);
  prof_end(t, c.s);
  return st;
}

extern "C" int vrs_linear_cross_entropy_backward_with_loss(
    const float* dloss, const void* x, int64_t x_stride, int64_t rows, const void* table, int64_t table_stride,
    int64_t classes, int64_t d, int32_t dtype, const int64_t* targets, float scale, const float* lse, const float* loss,
    void* dx, int64_t dx_stride, void* dtable, int64_t dtable_stride, void* workspace, int64_t workspace_bytes,
    void* cuda_stream) {
  using namespace vrs;
  using namespace vrs::ops;
  const std::string who = "vrs_linear_cross_entropy_backward";
  VRS_TRY(check(who, rows, classes, d, dtype));
  VRS_TRY(check_scale(who, scale));
  if ((rows > 1 && (x_stride < d || (dx && dx_stride < d))) ||
      (classes > 1 && (table_stride < d || (dtable && dtable_stride < d))))
    return invalid(who + ": row strides must be at least d");
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (rows == 0) {  // sums over no rows
    if (dtable)
      VRS_CUDA(cudaMemset2DAsync(dtable, (size_t)(classes > 1 ? dtable_stride : d) * 2, 0, (size_t)d * 2,
                                 (size_t)classes, s));
    return VRS_OK;
  }
  if (!dx && !dtable) return VRS_OK;
  if (!dloss || !x || !table || !targets || !lse) return invalid(who + ": null buffer");
  const Plan p = make_plan(rows, classes, d, true, tma_rows(table, table_stride, classes));
  VRS_TRY(check_workspace(who, workspace, workspace_bytes, p.bytes));
  const Call c{x, x_stride, rows, table, table_stride, classes, d, dtype, targets, scale, (char*)workspace, s};
  ProfToken t = prof_begin("linear_cross_entropy_backward", s);
  const int st = backward(c, p, dloss, lse, loss, dx, dx_stride, dtable, dtable_stride);
  prof_end(t, s);
  return st;
}

extern "C" int vrs_linear_cross_entropy_backward(const float* dloss, const void* x, int64_t x_stride, int64_t rows,
                                                 const void* table, int64_t table_stride, int64_t classes, int64_t d,
                                                 int32_t dtype, const int64_t* targets, float scale, const float* lse,
                                                 void* dx, int64_t dx_stride, void* dtable, int64_t dtable_stride,
                                                 void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  return vrs_linear_cross_entropy_backward_with_loss(dloss, x, x_stride, rows, table, table_stride, classes, d, dtype,
                                                     targets, scale, lse, nullptr, dx, dx_stride, dtable, dtable_stride,
                                                     workspace, workspace_bytes, cuda_stream);
}
