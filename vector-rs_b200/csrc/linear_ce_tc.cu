// linear_ce_tc.cu -- the matrix products of the linear cross entropy on
// tcgen05, CTA pairs (cta_group::2), one persistent kernel in three modes:
//   scores   z = x w^T      A = rows x d, B = classes x d, both K-major
//   dx       = g w          A = g (rows x classes) K-major, B = table MN-major
//   dtable   = g^T x        A = g MN-major, B = rows MN-major
// The transposed operands need no transposed copies: the tiles that TMA
// writes are read by the tensor cores as K-major or MN-major, whichever the
// product wants, by descriptor alone.
//
// A pair owns a tile of 256 rows (128 a CTA: its TMEM lanes) by up to 256
// columns; each CTA loads its half of both operands, 64 deep, into a ring of
// stages. One thread of the even CTA issues M = 256 MMAs into one of two
// accumulators (2 x 256 columns = all of TMEM). Two groups of epilogue warps a
// CTA (TMEM lane quadrant x the tile's columns, or half of them) take alternate
// tiles and read 32 columns ahead, so that one tile is exponentiated or stored
// while the other accumulator is written. The gradient of the scores leaves
// through swizzled staging tiles and TMA stores; the products, whose rows may
// start anywhere, through staging tiles that a warp reads back by whole lines,
// dx adding in f32 to what earlier pieces of the classes left.
//
// A row's target takes no part in the sums here, and its gradient is handed in:
// its score comes from dot_rows, which says why.
//
// Bound by the tensor cores for d of some hundreds and more; by the
// exponentials for small d (one a score, 16 an SM and clock, against
// 4,096 multiply-adds an SM and clock: equal at d = 256).
#include <atomic>

#include "linear_ce.cuh"
#include "tc_common.cuh"

namespace vrs {
namespace ops {
namespace {

using namespace vrs::tc;

constexpr int EPI_FIRST = 4;          // producer of A, MMA, TMEM, producer of B
// Epilogue warps: the scores' exponentials keep 16 busy (1,024 x 300,000 x 128:
// forward 121 us, with 8 of twice the columns 151 us); storing products takes 8.
constexpr int epi_warps(int mode) { return mode == kCeStore ? 8 : 16; }
constexpr int threads(int mode) { return 32 * (EPI_FIRST + epi_warps(mode)); }
constexpr int CHUNK = 32;             // columns that an epilogue warp loads at a time
constexpr int PART = 128;             // columns of one maximum and sum of the scores
constexpr int kTileCost = 4;          // of a tile beside its K blocks, in K blocks
constexpr uint32_t BOX = 64 * 128;    // bytes of a 64 x 64 tile of 16-bit operands
// A CTA's A, 128 x 64, and its half of B, 128 x 64, or without a partner all 256 x 64.
constexpr uint32_t stage_bytes(bool pair) { return (pair ? 4 : 6) * BOX; }
constexpr uint32_t STG = 32 * 128;    // a warp's staging tile: 32 rows of 128 bytes
constexpr size_t SMEM_BAR = 512;
constexpr uint64_t WAIT_NS = 2000000000ull;

constexpr int stages(int mode, bool pair) { return pair ? mode == kCeGrad ? 5 : 6 : mode == kCeGrad ? 3 : 4; }
constexpr size_t smem_bytes(int mode, bool pair) {
  return 1024 + (size_t)stages(mode, pair) * stage_bytes(pair) + (mode == kCeLse ? 0 : epi_warps(mode) * STG) + SMEM_BAR;
}
static_assert(smem_bytes(kCeLse, true) <= 232448 && smem_bytes(kCeGrad, true) <= 232448 &&
                  smem_bytes(kCeStore, true) <= 232448 && smem_bytes(kCeLse, false) <= 232448 &&
                  smem_bytes(kCeGrad, false) <= 232448,
              "above the per-block limit");

// ------------------------------------------------------------ PTX wrappers

// MN-major operand, 128-byte swizzle, as a TMA box of 64 (MN) x 64 (K)
// leaves it: 8 K-rows of 128 bytes form a 1,024-byte atom; the next 8 K-rows
// follow it (stride), the next 64 of MN start a box later (leading).
__device__ __forceinline__ uint64_t desc_mn(const void* p) {
  uint64_t d = smem_desc_sw128(p);
  d &= ~((uint64_t)0x3FFF << 16);
  d |= (uint64_t)(BOX >> 4) << 16;
  return d;
}

// A load that completes on a barrier of the pair's even CTA, or of this CTA.
template <bool PAIR>
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (PAIR) {
    tma_load_2d_pair(dst, map, x, y, bar);
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  }
}
template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    mma_f16_pair(d, ad, bd, idesc, accumulate);
  else
    mma_f16(d, ad, bd, idesc, accumulate);
}
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (PAIR)
    mma_commit_pair(bar, 0x3);
  else
    mma_commit(bar);
}
template <bool PAIR>
__device__ __forceinline__ void sync_all() {
  if (PAIR)
    cluster_sync();
  else
    __syncthreads();
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void add_f32x4(float* to, uint4 v) {
  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(__uint_as_float(v.x)),
               "f"(__uint_as_float(v.y)), "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w))
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 lanes x 32 columns; the values may be used only after tmem_wait.
__device__ __forceinline__ void tmem_ld_issue(uint32_t taddr, float (&v)[CHUNK]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
// The values pass through the wait, so no use of them can move before it.
__device__ __forceinline__ void tmem_wait(float (&v)[CHUNK]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---------------------------------------------------------------- the tiles

struct Tile {
  int job;         // kCeStore: 0 dx, 1 dtable
  int m, n, bn;    // tile row, first column (in elements) and columns
  int kb0, kb1;    // K blocks
  int split;
};

// Rows that take part: counted by the pack kernel, or all rows where no
// packing was needed.
__device__ __forceinline__ int taken_rows(const CeGemm& a) { return a.rows >= 0 ? a.rows : a.head->taken; }

// Bytes of the A operand that a CTA loads a stage in the score modes: with one
// tile of rows, those that hold rows. The others are zeroed once.
__device__ __forceinline__ uint32_t a_bytes(const CeGemm& a, int cta) {
  if (!a.one_tile_rows) return 2 * BOX;
  if (cta) return a.one_tile_rows > 128 ? 2 * BOX : 0;
  return a.one_tile_rows > 64 ? 2 * BOX : BOX;
}

struct Tiles {
  int mtiles;         // rows that take part, in tiles
  int kblocks_rows;   // and in K blocks
  int total;
  // Order of work in kCeStore: the product with the longer tiles (`job`)
  // first, one of its tiles as long as `ratio` of the other's.
  int long_job, n_long, n_short, ratio;
};

// A taking row's target; -1 for an unpacked row that takes no part.
__device__ __forceinline__ int target_of(const CeGemm& a, int64_t row) {
  if (!a.targets) return a.target[row];
  const int64_t t = a.targets[row];
  return t >= 0 && t < a.classes ? (int)t : -1;
}

template <int MODE>
__device__ __forceinline__ Tiles count_tiles(const CeGemm& a) {
  Tiles t;
  const int rows = taken_rows(a);
  t.mtiles = (rows + kCeM - 1) / kCeM;
  t.kblocks_rows = (rows + kCeK - 1) / kCeK;
  t.long_job = t.n_long = t.n_short = 0;
  t.ratio = 1;
  if (MODE == kCeStore) {
    const int n_dx = a.dx.on ? t.mtiles * a.dx.ntiles * a.dx.splits : 0;
    const int n_dw = a.dw.on ? a.dw.mtiles * a.dw.ntiles * a.dw.splits : 0;
    const int k_dx = (a.dx.planes * a.dx.kblocks + a.dx.splits - 1) / a.dx.splits + kTileCost;
    const int k_dw = (a.dw.planes * t.kblocks_rows + a.dw.splits - 1) / a.dw.splits + kTileCost;
    t.long_job = k_dw > k_dx;
    t.n_long = t.long_job ? n_dw : n_dx;
    t.n_short = t.long_job ? n_dx : n_dw;
    t.ratio = max(1, t.long_job ? (k_dw + k_dx / 2) / k_dx : (k_dx + k_dw / 2) / k_dw);
    t.total = n_dx + n_dw;
  } else {
    t.total = t.mtiles * a.vtiles;
  }
  return t;
}

// The i-th tile of a pair, -1 past its last. Scores: every npairs-th. Products:
// the long tiles first, in turn; the pairs that the last turn of them leaves
// out take `ratio` short ones meanwhile; the rest of those in turn.
template <int MODE>
__device__ __forceinline__ int nth_tile(const Tiles& c, int i, int pair, int npairs) {
  if (MODE != kCeStore) {
    const int id = pair + i * npairs;
    return id < c.total ? id : -1;
  }
  const int rem = c.n_long % npairs;
  const int mine = c.n_long / npairs + (pair < rem);
  if (i < mine) return pair + i * npairs;
  i -= mine;
  const int free_pairs = rem ? npairs - rem : 0;
  int j;
  if (free_pairs && pair >= rem && i < c.ratio)
    j = i * free_pairs + pair - rem;
  else
    j = free_pairs * c.ratio + (i - (free_pairs && pair >= rem ? c.ratio : 0)) * npairs + pair;
  return j < c.n_short ? c.n_long + j : -1;
}

// By value, field by field: a reference chosen at run time would read the
// kernel's parameters through memory, again after every asm statement.
__device__ __forceinline__ CeJob job_of(const CeGemm& a, bool dw) {
  CeJob j;
  j.mtiles = dw ? a.dw.mtiles : a.dx.mtiles;
  j.ntiles = dw ? a.dw.ntiles : a.dx.ntiles;
  j.kblocks = dw ? a.dw.kblocks : a.dx.kblocks;
  j.splits = dw ? a.dw.splits : a.dx.splits;
  j.planes = dw ? a.dw.planes : a.dx.planes;
  j.f32 = dw ? a.dw.f32 : a.dx.f32;
  j.f32_rows = dw ? a.dw.f32_rows : a.dx.f32_rows;
  j.add = dw ? a.dw.add : a.dx.add;
  j.row0 = dw ? a.dw.row0 : a.dx.row0;
  j.out = dw ? a.dw.out : a.dx.out;
  j.out_stride = dw ? a.dw.out_stride : a.dx.out_stride;
  j.out_vec = dw ? a.dw.out_vec : a.dx.out_vec;
  return j;
}

template <int MODE>
__device__ __forceinline__ Tile tile_at(const CeGemm& a, const Tiles& c, int id) {
  Tile t;
  if (MODE != kCeStore) {
    // Row tiles first: the pairs that run together share few class tiles,
    // and the rows' operand stays in L2.
    t.job = 0;
    t.m = id % c.mtiles;
    const int n = id / c.mtiles;
    t.bn = n < a.whole ? kCeN : kCeN / 2;
    t.n = n < a.whole ? n * kCeN : a.whole * kCeN + (n - a.whole) * (kCeN / 2);
    t.kb0 = 0;
    t.kb1 = a.kblocks;
    t.split = 0;
    return t;
  }
  const bool second = id >= c.n_long;
  t.job = second ? !c.long_job : c.long_job;
  if (second) id -= c.n_long;
  const CeJob j = job_of(a, t.job);
  t.n = id % j.ntiles * kCeN;
  id /= j.ntiles;
  t.split = id % j.splits;
  t.m = id / j.splits;
  t.bn = a.d - t.n > 128 ? 256 : 128;
  const int kb = j.planes * (t.job ? c.kblocks_rows : j.kblocks);
  const int per = (kb + j.splits - 1) / j.splits;
  t.kb0 = min(kb, t.split * per);
  t.kb1 = min(kb, t.kb0 + per);
  return t;
}

// --------------------------------------------------------------- epilogues

// 32 scores of a row: the running maximum and sum of powers of two (the scores
// times scale * log2(e), so that e^z is one ex2). The target's own score is
// left out: the combining kernel computes it apart.
__device__ __forceinline__ void epi_lse(const CeGemm& a, float (&w)[CHUNK], int n0, int cols, int tgt, float& top,
                                        float& sum) {
  if (cols <= 0) return;
  if (cols < CHUNK) {
#pragma unroll
    for (int j = 0; j < CHUNK; j++)
      if (j >= cols) w[j] = -INFINITY;
  }
  const int at = tgt - n0;
  if (at >= 0 && at < CHUNK) {
#pragma unroll
    for (int j = 0; j < CHUNK; j++)
      if (j == at) w[j] = -INFINITY;
  }
  float m[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    m[k] = fmax3(w[16 * k], w[16 * k + 1], w[16 * k + 2]);
#pragma unroll
    for (int j = 3; j < 15; j += 2) m[k] = fmax3(m[k], w[16 * k + j], w[16 * k + j + 1]);
    m[k] = fmaxf(m[k], w[16 * k + 15]);
  }
  const float now = fmaxf(m[0], m[1]) * a.c2;
  if (now > top) {
    sum *= ex2(top - now);
    top = now;
  }
  const float sub = top == -INFINITY ? 0.0f : top;
  F2 s[2] = {pack_f2(0.0f), pack_f2(0.0f)};
  const F2 cc = pack_f2(a.c2), dd = pack_f2(-sub);
#pragma unroll
  for (int q = 0; q < CHUNK / 2; q++) {
    float lo, hi;
    unpack_f2(fma2(pack_f2(w[2 * q], w[2 * q + 1]), cc, dd), lo, hi);
    s[q & 1] = add2(s[q & 1], pack_f2(ex2(lo), ex2(hi)));
  }
  sum += sum_f2(add2(s[0], s[1]));
}

// A staging tile is free again once its last store has read it.
__device__ __forceinline__ void stage_ready(int lane) {
  if (lane == 0) bulk_wait_read<0>();
  __syncwarp();
}

// Row `lane` of a staging tile: 16-byte chunk j, 128-byte swizzle.
__device__ __forceinline__ void stage_put(uint8_t* stg, int lane, int j, uint4 q) {
  *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = q;
}

__device__ __forceinline__ uint4 stage_get(const uint8_t* stg, int row, int j) {
  return *reinterpret_cast<const uint4*>(stg + row * 128 + ((j ^ (row & 7)) << 4));
}

// Rows first, first + STEP, ... (first < STEP) of a staging tile of 16-bit
// values to rows that start on (ODD: between) 4-byte words; `here` of their 64
// elements. Between words a lane's word holds elements of two lanes, and the
// first and the last element go by themselves.
template <int ODD, int STEP>
__device__ __forceinline__ void store_rows(uint16_t* o, int64_t pitch, const uint8_t* stg, int first, int all,
                                           int here, int lane) {
  const int e = 2 * lane;
  uint16_t* to = o + first * pitch + e;
  pitch *= STEP;
  auto word_of = [&](int r, int i) {
    return *reinterpret_cast<const uint32_t*>(
        stg + (r + i * STEP) * 128 + (((lane >> 2) ^ ((first + i * STEP) & 7)) << 4 | (lane & 3) << 2));
  };
  if (all == 32 && here >= 64) {  // whole tiles: fewer instructions a row
    const int edge = lane ? 1 : 0;  // the element that lane 0 or 31 stores by itself
    const bool word = !ODD || lane < 31, one = ODD && (lane == 0 || lane == 31);
#pragma unroll 1
    for (int r = first; r < 32; r += 8 * STEP) {
      uint32_t k[8], w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) k[i] = word_of(r, i);
#pragma unroll
      for (int i = 0; i < 8; i++) w[i] = ODD ? __funnelshift_r(k[i], __shfl_down_sync(~0u, k[i], 1), 16) : k[i];
      if (word) {
        uint16_t* q = to + ODD;
#pragma unroll
        for (int i = 0; i < 8; i++, q += pitch) *reinterpret_cast<uint32_t*>(q) = w[i];
      }
      if (one) {
        uint16_t* q = to + edge;
#pragma unroll
        for (int i = 0; i < 8; i++, q += pitch) *q = (uint16_t)(k[i] >> 16 * edge);
      }
      to += 8 * pitch;
    }
    return;
  }
  const bool whole = ODD ? lane < 31 && e + 2 < here : e + 1 < here;
  const bool low = ODD ? lane == 0 : e + 1 == here;
  const bool high = ODD && (e + 2 == here || (lane == 31 && here >= 64));
#pragma unroll 1
  for (int r = first; r < all; r += 8 * STEP) {
    uint32_t k[8], word[8];
#pragma unroll
    for (int i = 0; i < 8; i++) k[i] = word_of(r, i);  // eight reads in flight, none past the tile's 32 rows
#pragma unroll
    for (int i = 0; i < 8; i++) word[i] = ODD ? __funnelshift_r(k[i], __shfl_down_sync(~0u, k[i], 1), 16) : k[i];
#pragma unroll
    for (int i = 0; i < 8; i++, to += pitch) {
      const bool in = r + i * STEP < all;
      if (in && whole) *reinterpret_cast<uint32_t*>(to + ODD) = word[i];
      if (in && low) *to = (uint16_t)k[i];
      if (ODD && in && high) to[1] = (uint16_t)(k[i] >> 16);
    }
  }
}

// 32 values of a row in 16 bits into one half of the staging tile.
template <bool F16>
__device__ __forceinline__ void stage_row16(uint8_t* stg, int lane, int half, const float (&w)[CHUNK]) {
#pragma unroll
  for (int q = 0; q < 4; q++)
    stage_put(stg, lane, half * 4 + q,
              make_uint4(pack2<F16>(w[8 * q], w[8 * q + 1]), pack2<F16>(w[8 * q + 2], w[8 * q + 3]),
                         pack2<F16>(w[8 * q + 4], w[8 * q + 5]), pack2<F16>(w[8 * q + 6], w[8 * q + 7])));
}

// What rounding to 16 bits leaves of 32 values, itself rounded.
template <bool F16>
__device__ __forceinline__ void store_rest(uint16_t* to, const float (&w)[CHUNK]) {
#pragma unroll
  for (int q = 0; q < CHUNK / 8; q++) {
    uint32_t k[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float lo = w[8 * q + 2 * i], hi = w[8 * q + 2 * i + 1];
      const uint32_t u = pack2<F16>(lo, hi);
      const float rl = F16 ? __half2float(__ushort_as_half(u & 0xffff)) : __uint_as_float(u << 16);
      const float rh = F16 ? __half2float(__ushort_as_half(u >> 16)) : __uint_as_float(u & 0xffff0000u);
      k[i] = pack2<F16>(lo - rl, hi - rh);
    }
    *reinterpret_cast<uint4*>(to + 8 * q) = make_uint4(k[0], k[1], k[2], k[3]);
  }
}

// ------------------------------------------------------------------ kernel

// PAIR: as the head of this file says. Else, scores of up to 128 rows: a CTA by
// itself, M = 128, takes tiles of its own; a partner would multiply zeros, and
// these calls wait for the table to come from memory.
template <int MODE, bool F16, bool PAIR>
__global__ void __launch_bounds__(threads(MODE), 1)
    ce_gemm_kernel(const __grid_constant__ CeMaps maps, const __grid_constant__ CeGemm a) {
  constexpr int ST = stages(MODE, PAIR), EW = epi_warps(MODE);
  constexpr uint32_t STAGE = stage_bytes(PAIR);
  constexpr int HCOLS = 2048 / EW;  // columns of an epilogue warp: the tile's or half of them
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_stg = smem + (size_t)ST * STAGE;
  uint64_t* bars = (uint64_t*)(s_stg + (MODE == kCeLse ? 0 : EW * STG));
  uint64_t* full = bars;           // [ST] even CTA: both CTAs' bytes
  uint64_t* empty = full + ST;     // [ST] each CTA: MMA commit
  uint64_t* tfull = empty + ST;    // [2] each CTA: MMA commit
  uint64_t* tempty = tfull + 2;    // [2] even CTA: both CTAs' epilogue warps
  uint32_t* s_tmem = (uint32_t*)(tempty + 2);
  volatile int* s_abort = (volatile int*)(s_tmem + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = PAIR ? (int)cluster_ctarank() : 0;
  const bool lead = cta == 0;
  const int pair = PAIR ? blockIdx.x >> 1 : blockIdx.x, npairs = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], PAIR ? EW : EW / 2);  // half of a CTA's take the buffer's tiles
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  if (threadIdx.x == 32 * 3) {
    prefetch_tmap(&maps.a0);
    prefetch_tmap(&maps.b0);
    if (MODE == kCeStore) {
      prefetch_tmap(&maps.a1);
      prefetch_tmap(&maps.b1);
    }
    if (MODE == kCeGrad) prefetch_tmap(&maps.out0);
  }
  if (warp == 2) {
    if (PAIR)
      tmem_alloc_pair(s_tmem, 512);
    else
      tmem_alloc(s_tmem, 512);
  }
  if (MODE != kCeStore && a.one_tile_rows) {
    const int skip = (int)a_bytes(a, cta);
    for (int s = 0; s < ST; s++)
      for (int i = skip + (int)threadIdx.x * 16; i < 2 * (int)BOX; i += threads(MODE) * 16)
        *reinterpret_cast<uint4*>(smem + s * STAGE + i) = make_uint4(0, 0, 0, 0);
    fence_async_smem();
  }
  tc_fence_before();
  sync_all<PAIR>();  // barriers initialised and TMEM allocated in both CTAs
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // The set-up above overlaps the end of the kernel before; its results are
  // there from here on.
  grid_launch();
  grid_wait();
  const Tiles cnt = count_tiles<MODE>(a);

  if (warp == 0 || warp == 3) {
    // ---------------------------------------------------- TMA producers
    // One thread issues a K block's A loads, one its B loads: a K block lasts
    // 512 clocks, which one thread for all of them did not always meet.
    if (lane == 0) {
      const bool for_a = warp == 0;
      const uint32_t full0 = PAIR ? mapa_shared(full, 0) : smem_u32(full);
      const uint32_t bytes_a = MODE == kCeStore ? 4 * BOX : a_bytes(a, 0) + a_bytes(a, 1);
      const bool load_a = MODE == kCeStore || a_bytes(a, cta) > 0;
      int s = 0, it = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int i = 0, id; ok && (id = nth_tile<MODE>(cnt, i, pair, npairs)) >= 0; i++) {
        const Tile t = tile_at<MODE>(a, cnt, id);
        const int ra = t.m * kCeM + cta * 128;
        const int boxes = PAIR ? t.bn >> 7 : t.bn >> 6;  // of 64 columns of B in each CTA
        const int rb = t.n + cta * boxes * 64;
        const bool two = boxes == 2;
        const uint32_t bytes = bytes_a + (t.bn >> 6) * BOX;
        const CUtensorMap* map = for_a ? (MODE == kCeStore && t.job ? &maps.a1 : &maps.a0)
                                       : (MODE == kCeStore && t.job ? &maps.b1 : &maps.b0);
        const int v0 = MODE == kCeStore && t.job ? 0 : a.v0;
        for (int kb = t.kb0; kb < t.kb1; kb++, it++) {
          if (!mbar_wait(&empty[s], phase, s_abort, a.err, 31, WAIT_NS)) {
            ok = false;
            break;
          }
          uint8_t* to = smem + s * STAGE;
          const uint32_t bar = full0 + s * 8;
          int k = kb * kCeK, plane = 0;
          if (MODE == kCeStore) {
            const int kb_plane = t.job ? cnt.kblocks_rows : a.dx.kblocks;
            if (kb >= kb_plane) {  // the second plane, against the same rows or classes
              k -= kb_plane * kCeK;
              plane = a.plane_rows;
            }
          }
          if (for_a) {
            if (lead) mbar_expect_tx(&full[s], bytes);
            if (MODE != kCeStore) {
              if (load_a) tma_load<PAIR>(to, map, k, ra, bar);
            } else if (t.job == 0) {
              tma_load_2d_pair(to, map, k, plane + ra, bar);
            } else {
              tma_load_2d_pair(to, map, ra, plane + k, bar);
              tma_load_2d_pair(to + BOX, map, ra + 64, plane + k, bar);
            }
          } else {
            if (MODE != kCeStore) {
              for (int i = 0; i < boxes; i++) tma_load<PAIR>(to + (2 + i) * BOX, map, k, v0 + rb + 64 * i, bar);
            } else {
              tma_load_2d_pair(to + 2 * BOX, map, rb, v0 + k, bar);
              if (two) tma_load_2d_pair(to + 3 * BOX, map, rb + 64, v0 + k, bar);
            }
          }
          if (++s == ST) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      if (*s_abort && lead && for_a) {
        // Drain (bounded): both CTAs' loads complete on these barriers.
        volatile int dummy = 0;
        for (int i = max(0, it - ST); i < it; i++)
          mbar_wait(&full[i % ST], (i / ST) & 1, &dummy, a.err, 0, WAIT_NS / 4);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------- MMA issuer (even CTA)
    if (lane == 0 && lead) {
      // Descriptors of stage 0, K-major and MN-major (shared addresses are
      // below 2^18: adding 16-byte units does not carry out of the field).
      const uint64_t ka = smem_desc_sw128(smem), kb_ = smem_desc_sw128(smem + 2 * BOX);
      const uint64_t ma = desc_mn(smem), mb = desc_mn(smem + 2 * BOX);
      int s = 0, tn = 0, last = -1;
      uint32_t phase = 0;
      bool ok = true;
      for (int id; ok && (id = nth_tile<MODE>(cnt, tn, pair, npairs)) >= 0; tn++) {
        const Tile t = tile_at<MODE>(a, cnt, id);
        const int b = tn & 1;
        if (!mbar_wait(&tempty[b], ((tn >> 1) & 1) ^ 1, s_abort, a.err, 32, WAIT_NS)) break;
        tc_fence_after();
        // (A split without K blocks commits at once: its epilogue stores zeros.)
        const uint32_t d = tmem + b * 256;
        const bool a_mn = MODE == kCeStore && t.job == 1, b_mn = MODE == kCeStore;
        const uint32_t idesc = a.idesc | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(t.bn >> 3) << 17) |
                               ((PAIR ? 256u : 128u) >> 4 << 24);
        const uint64_t ad0 = a_mn ? ma : ka, bd0 = b_mn ? mb : kb_;
        // 16 of K: 32 bytes on in a K-major row, 16 rows on in an MN-major box.
        const uint32_t astep = a_mn ? 2048 >> 4 : 32 >> 4, bstep = b_mn ? 2048 >> 4 : 32 >> 4;
        for (int kb = t.kb0; kb < t.kb1; kb++) {
          if (!mbar_wait(&full[s], phase, s_abort, a.err, 33, WAIT_NS)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = ad0 + s * (STAGE >> 4), bd = bd0 + s * (STAGE >> 4);
#pragma unroll
          for (int ks = 0; ks < 4; ks++)
            mma<PAIR>(d, ad + ks * astep, bd + ks * bstep, idesc, kb > t.kb0 || ks > 0 ? 1u : 0u);
          commit<PAIR>(&empty[s]);
          if (++s == ST) {
            s = 0;
            phase ^= 1;
          }
        }
        commit<PAIR>(&tfull[b]);
        last = tn;
      }
      if (*s_abort && last >= 0) {
        volatile int dummy = 0;
        mbar_wait(&tfull[last & 1], (last >> 1) & 1, &dummy, a.err, 0, WAIT_NS / 4);
      }
    }
  } else if (warp >= EPI_FIRST) {
    // ---------------------------------------------------- epilogue
    const int ew = warp - EPI_FIRST, group = ew / (EW / 2), half = ew / 4 % (EW / 8), quad = warp & 3;
    uint8_t* stg = s_stg + ew * STG;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + group * 256 + half * HCOLS;
    const int taken = taken_rows(a);
    int tn = 0;
    for (int id; (id = nth_tile<MODE>(cnt, tn, pair, npairs)) >= 0; tn++) {
      if ((tn & 1) != group) continue;
      const Tile t = tile_at<MODE>(a, cnt, id);
      const int r0 = t.m * kCeM + cta * 128 + quad * 32;  // the warp's first row
      const int64_t row = r0 + lane;
      const int n0 = t.n + half * HCOLS;                  // and column
      const bool live = row < taken;
      int tgt = -1;
      float lse2 = 0.0f, gs = 0.0f, gy = 0.0f;
      if (MODE != kCeStore && live) {
        tgt = target_of(a, row);
        if (MODE == kCeGrad) {
          lse2 = a.lse2[row];
          gs = a.gs[row];
          gy = a.gy[row];
        }
      }
      const bool ok = mbar_wait(&tfull[group], (tn >> 1) & 1, s_abort, a.err, 34, WAIT_NS);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      // Columns of the warp that exist: the last class or a dx or dtable row may
      // end within the tile.
      const int cols = min(t.bn - half * HCOLS, (MODE == kCeStore ? a.d : MODE == kCeGrad ? a.vn : a.classes) - n0);
      // Rows that exist; of the score gradients, those in dtable's last K block too.
      const bool rows = MODE == kCeLse ? r0 < taken : MODE == kCeGrad ? r0 < (taken + kCeK - 1) / kCeK * kCeK : true;
      const bool mine = half * HCOLS < t.bn && rows && (MODE == kCeGrad || cols > 0);
      const CeJob job = job_of(a, t.job);
      const bool none = MODE == kCeStore && t.kb0 == t.kb1;  // a split without K blocks: zeros
      const float f = MODE == kCeStore ? a.head->grad_scale : 1.0f;
      float top = -INFINITY, sum = 0.0f;
      float v[2][CHUNK];
      if (mine) tmem_ld_issue(taddr, v[0]);
      // Two chunks a turn (one read ahead of the other) and no more unrolling:
      // in a small problem this code runs once, and its fetch would show.
#pragma unroll 1
      for (int c0 = 0; c0 < HCOLS / CHUNK; c0 += 2)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int c = c0 + h;
        float(&w)[CHUNK] = v[h];
        if (mine) tmem_wait(w);
        if (c + 1 < HCOLS / CHUNK) {
          if (mine) tmem_ld_issue(taddr + (c + 1) * CHUNK, v[1 - h]);
        } else {
          // The last columns are in registers: hand the accumulator back.
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (lead)
              mbar_arrive(&tempty[group]);
            else
              mbar_arrive_cluster(mapa_shared(&tempty[group], 0));
          }
        }
        if (!mine) continue;
        const int left = cols - c * CHUNK;
        if (MODE == kCeLse) {
          epi_lse(a, w, n0 + c * CHUNK, left, tgt, top, sum);
          if ((c + 1) * CHUNK % PART == 0) {
            // Neighbouring lanes (rows) side by side.
            const int part = (n0 + c * CHUNK) / PART;
            if (live && left + PART - CHUNK > 0) a.part[(int64_t)part * a.part_rows + row] = make_float2(top, sum);
            top = -INFINITY;
            sum = 0.0f;
          }
        } else if (MODE == kCeGrad) {
          // g = (2^(c2 z - lse2) - [target]) gs in 16 bits; zeros past the last
          // class and in the rest of the last K block of rows. (dx's product reads
          // the whole tile of rows; what those further down hold reaches rows of its
          // result that nobody reads.)
#pragma unroll
          for (int j = 0; j < CHUNK; j++) w[j] = ex2(fmaf(w[j], a.c2, -lse2));
          const int at = tgt - a.v0 - n0 - c * CHUNK;
          if (at >= 0 && at < CHUNK) {
#pragma unroll
            for (int j = 0; j < CHUNK; j++)
              if (j == at) w[j] = gy;
          }
#pragma unroll
          for (int j = 0; j < CHUNK; j++) w[j] *= gs;
          if (left < CHUNK || !live) {
#pragma unroll
            for (int j = 0; j < CHUNK; j++)
              if (!live || j >= left) w[j] = 0.0f;
          }
          if (a.planes > 1) store_rest<F16>(a.g + (a.plane_rows + row) * a.g_pitch + n0 + c * CHUNK, w);
          if (h == 0) stage_ready(lane);
          stage_row16<F16>(stg, lane, h, w);
          if (h == 1) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&maps.out0, stg, n0 + (c - 1) * CHUNK, r0);
              bulk_commit();
            }
          }
        } else {
          if (none) {
#pragma unroll
            for (int i = 0; i < CHUNK; i++) w[i] = 0.0f;
          }
          if (job.f32) {
            // Through the staging tile, so that a warp's store covers whole
            // lines. Whole tiles of rows: never past the end of the split's
            // result. Each value has one writer a launch, so additions come in
            // launch order.
#pragma unroll
            for (int q = 0; q < CHUNK / 4; q++)
              stage_put(stg, lane, q,
                        make_uint4(__float_as_uint(w[4 * q]), __float_as_uint(w[4 * q + 1]),
                                   __float_as_uint(w[4 * q + 2]), __float_as_uint(w[4 * q + 3])));
            __syncwarp();
            float* o = job.f32 + (t.split * (int64_t)job.f32_rows + r0) * a.d4 + n0 + c * CHUNK;
            const int col = (lane & 7) * 4;
#pragma unroll
            for (int q = 0; q < 8; q++) {
              const int r = q * 4 + (lane >> 3);
              const uint4 k = stage_get(stg, r, lane & 7);
              if (col < left) {
                if (job.add)
                  add_f32x4(o + (int64_t)r * a.d4 + col, k);
                else
                  *reinterpret_cast<uint4*>(o + (int64_t)r * a.d4 + col) = k;
              }
            }
            __syncwarp();
          } else {
            if (left + h * CHUNK <= 0) continue;  // the 64 columns of a staging tile
#pragma unroll
            for (int i = 0; i < CHUNK; i++) w[i] *= f;
            stage_row16<F16>(stg, lane, h, w);
            if (h == 0) continue;
            __syncwarp();
            const int64_t first = job.row0 + (int64_t)r0, past = a.classes - first;
            uint16_t* o = job.out + first * job.out_stride + n0 + c0 * CHUNK;
            const int here = left + CHUNK;  // of the staging tile's 64 columns
            if (job.out_vec) {
              const int col = (lane & 7) * 8;
#pragma unroll
              for (int q = 0; q < 8; q++) {
                const int r = q * 4 + (lane >> 3);
                const uint4 k = stage_get(stg, r, lane & 7);
                if (r < past && col < here) *reinterpret_cast<uint4*>(o + r * job.out_stride + col) = k;
              }
            } else {
              // Rows that 16-byte stores cannot address: a word a lane, the rows
              // that start on a word and the others apart. Few warps store, so
              // the instructions and latencies of a row count (10 x 150,379 x
              // 798, 120 M elements of dtable: 198 us; element by element 346).
              const int all = (int)min((int64_t)32, past);
              const int odd = (int)(reinterpret_cast<uintptr_t>(o) >> 1 & 1);
              if ((job.out_stride & 1) == 0) {
                if (odd)
                  store_rows<1, 1>(o, job.out_stride, stg, 0, all, here, lane);
                else
                  store_rows<0, 1>(o, job.out_stride, stg, 0, all, here, lane);
              } else {
                store_rows<0, 2>(o, job.out_stride, stg, odd, all, here, lane);
                store_rows<1, 2>(o, job.out_stride, stg, 1 - odd, all, here, lane);
              }
            }
            __syncwarp();
          }
        }
      }
    }
    if (MODE == kCeGrad && lane == 0) bulk_wait_read<0>();  // shared memory must stay until then
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // no MMA, load or remote arrival of either CTA is still pending
  if (warp == 2) {
    tc_fence_after();
    if (PAIR)
      tmem_dealloc_pair(tmem, 512);
    else
      tmem_dealloc(tmem, 512);
  }
}

// CTAs (or pairs) of the kernel that the current device runs at the same time,
// asked once per device, with the shared memory that it needs allowed.
template <int MODE, bool F16, bool PAIR>
int units_of(const cudaLaunchConfig_t& cfg, int* out) {
  static std::atomic<int> cached[128];
  int dev = 0;
  VRS_CUDA(cudaGetDevice(&dev));
  int n = dev < 128 ? cached[dev].load() : 0;
  if (n == 0) {
    auto kernel = ce_gemm_kernel<MODE, F16, PAIR>;
    VRS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(MODE, PAIR)));
    if (PAIR)
      VRS_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    else
      VRS_TRY(sm_count(&n));
    if (n < 1) {
      set_error(VRS_ERR_DRIVER, "linear cross entropy: no CTA pair of the product kernel fits this device");
      return VRS_ERR_DRIVER;
    }
    if (dev < 128) cached[dev].store(n);
  }
  *out = n;
  return VRS_OK;
}

template <int MODE, bool F16, bool PAIR>
int launch(const CeMaps& maps, const CeGemm& a, int64_t most_tiles, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(PAIR ? 2 : 1);
  cfg.blockDim = dim3(threads(MODE));
  cfg.dynamicSmemBytes = smem_bytes(MODE, PAIR);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = PAIR ? 2 : 1;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int units = 0;
  VRS_TRY((units_of<MODE, F16, PAIR>(cfg, &units)));
  const int64_t n = most_tiles < units ? most_tiles : units;
  cfg.gridDim = dim3((unsigned)((PAIR ? 2 : 1) * (n < 1 ? 1 : n)));
  cfg.numAttrs = 2;
  VRS_CUDA(cudaLaunchKernelEx(&cfg, ce_gemm_kernel<MODE, F16, PAIR>, maps, a));
  count_launch();
  return VRS_OK;
}

template <int MODE, bool PAIR>
int launch_type(bool is_f16, const CeMaps& maps, const CeGemm& a, int64_t most_tiles, cudaStream_t s) {
  return is_f16 ? launch<MODE, true, PAIR>(maps, a, most_tiles, s) : launch<MODE, false, PAIR>(maps, a, most_tiles, s);
}

}  // namespace

int launch_ce_gemm(int mode, bool is_f16, const CeMaps& maps, const CeGemm& a, int64_t most_tiles, cudaStream_t s) {
  const bool pair = !ce_single(a.one_tile_rows);
  switch (mode) {
    case kCeLse:
      return pair ? launch_type<kCeLse, true>(is_f16, maps, a, most_tiles, s)
                  : launch_type<kCeLse, false>(is_f16, maps, a, most_tiles, s);
    case kCeGrad:
      return pair ? launch_type<kCeGrad, true>(is_f16, maps, a, most_tiles, s)
                  : launch_type<kCeGrad, false>(is_f16, maps, a, most_tiles, s);
    default: return launch_type<kCeStore, true>(is_f16, maps, a, most_tiles, s);
  }
}

}  // namespace ops
}  // namespace vrs
