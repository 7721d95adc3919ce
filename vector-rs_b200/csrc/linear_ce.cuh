// linear_ce.cuh -- between the host plan of the linear cross entropy
// (linear_ce.cu) and its tensor-core products (linear_ce_tc.cu).
#pragma once
#include <cuda.h>

#include "ops_common.cuh"

namespace vrs {
namespace ops {

// A pair of CTAs computes tiles of 256 x 256 (or 256 x 128) over K blocks of 64.
constexpr int kCeM = 256;
constexpr int kCeN = 256;
constexpr int kCeK = 64;

// Written on the device by the first kernel of a call.
struct CeHeader {
  int taken;          // rows that take part
  float grad_scale;   // what the products of the score gradients are multiplied by
};

enum CeMode : int {
  kCeLse = 0,    // scores; each row's maximum and sum of e^(z - maximum) per class tile
  kCeGrad = 1,   // scores again; their gradient in 16 bits for one piece of the classes
  kCeStore = 2,  // the products of the score gradients: dx (rows x d), dtable (classes x d)
};

// One product of kCeStore. K is split over `splits` tiles with results of
// their own ([split][rows_out][d4], added later in split order).
struct CeJob {
  int on;
  int mtiles;      // dtable; dx takes its count from the header
  int ntiles;      // over d
  int kblocks;     // dx; dtable takes its count from the header
  int splits;
  int planes;      // of the score gradients that it takes
  float* f32;      // [split][f32_rows][d4], or null: 16-bit result, one split
  int f32_rows;
  int add;         // f32: add to what earlier pieces left
  int row0;        // 16-bit result: first row (the piece's first class)
  uint16_t* out;   // 16-bit result
  int64_t out_stride;
  int out_vec;     // its rows take 16-byte stores
};

struct CeGemm {
  const CeHeader* head;
  int rows;          // rows that take part, -1: head->taken
  int whole;         // tiles of 256 columns; those after them have 128 (kCeLse)
  int one_tile_rows; // scores: the rows where one tile holds them all, else 0
  int* err;          // host-visible word that a wait which gave up writes
  int classes;       // all classes
  int v0, vn;        // the piece
  int d, d4;         // d4: pitch of f32 results, d in whole fours
  int kblocks;       // of d
  int vtiles;        // class tiles of the piece
  int parts;         // kCeLse: 128-class parts of a row
  uint32_t idesc;    // types; majorness, M and N are added by the kernel
  // scores
  const int64_t* targets;  // [rows] where the rows are not packed, else null
  const int* target;       // [rows] of the taking rows
  const float* lse2;   // [rows] lse * log2(e)
  const float* gy;     // [rows] the target's probability - 1
  const float* gs;     // [rows] dloss over the largest finite |dloss| (f16: times a gain)
  float c2;            // scale * log2(e)
  int64_t part_rows;
  float2* part;        // [part][part_rows]: maximum of c2 z and sum of 2^(c2 z - maximum)
  float scale;
  const uint16_t* x;   // the rows and the table for the targets' scores, 16-byte aligned
  int64_t xs;
  const uint16_t* w;
  int64_t ws;
  // products
  CeJob dx, dw;
  int planes;          // of the score gradients written: 1, or 2 (rounded value, and what rounding left)
  int plane_rows;      // rows of a plane
  uint16_t* g;
  int64_t g_pitch;
};

// 2^x, the score exponentials' instruction.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The product of two rows of d 16-bit floats by one warp, rounded to nearest at
// every step. The tensor cores' sums are cut off instead: over d terms of one
// sign, as a trained row's product with its target has, some d / 16 half units
// of the last place, all downwards. A loss that is small against the target's
// score, and a probability near 1, would show them (2e-3 of the loss at
// d = 1,700), so the target's score is computed apart; another class's error is
// one of many. vec: both rows start on 16 bytes; the order of the sums is the same
// either way, so that both passes get one score from packed and unpacked rows.
template <bool F16>
__device__ __forceinline__ float dot_rows(const uint16_t* x, const uint16_t* w, int d, bool vec) {
  auto value = [](uint16_t u) {
    return F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float((uint32_t)u << 16);
  };
  const int lane = threadIdx.x & 31;
  float s[2] = {0.0f, 0.0f};
  int e = d / 8 * 8;  // first element of the tail
  for (int c = lane * 8; c < e; c += 256) {
    Pack<uint16_t, 8> p, q;
    if (vec) {
      p = load_pack<uint16_t, 8>(x + c);
      q = load_pack<uint16_t, 8>(w + c);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        p.v[j] = x[c + j];
        q.v[j] = w[c + j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) s[j & 1] = fmaf(value(p.v[j]), value(q.v[j]), s[j & 1]);
  }
  for (e += lane; e < d; e += 32) s[0] = fmaf(value(x[e]), value(w[e]), s[0]);
  float t = s[0] + s[1];
#pragma unroll
  for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// Tensor maps of a launch. Scores: a0 rows, b0 table, out0 their gradient.
// Products: a0, b0 of dx (A: the score gradients), a1, b1 of dtable.
struct CeMaps {
  CUtensorMap a0, b0, out0, a1, b1;
};

// Whether the score modes run on single CTAs (twice as many tiles at a time).
inline bool ce_single(int one_tile_rows) { return one_tile_rows > 0 && one_tile_rows <= 128; }

int launch_ce_gemm(int mode, bool is_f16, const CeMaps& maps, const CeGemm& a, int64_t most_tiles, cudaStream_t s);

}  // namespace ops
}  // namespace vrs
