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
  const float* gs;     // [rows] dloss over the largest |dloss| (f16: times a gain)
  float c2;            // scale * log2(e)
  int64_t part_rows;
  float2* part;        // [part][part_rows]: maximum of c2 z and sum of 2^(c2 z - maximum)
  float* zt;           // [row] c2 * target's score
  // products
  CeJob dx, dw;
};

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
