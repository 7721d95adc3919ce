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
// accumulators (2 x 256 columns = all of TMEM). Sixteen epilogue warps a CTA
// (TMEM lane quadrant x 64 columns) load a tile into registers and hand its
// accumulator back at once, so a tile is exponentiated and stored while the
// next two are multiplied. Results leave through swizzled staging tiles and
// TMA stores, in f32 also as TMA additions to what earlier pieces of the
// classes left.
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

constexpr int EPI_FIRST = 4;          // producer, MMA, TMEM, spare
constexpr int EPI_WARPS = 16;
constexpr int THREADS = 32 * (EPI_FIRST + EPI_WARPS);
constexpr int QCOLS = 64;             // columns of an epilogue warp
constexpr uint32_t BOX = 64 * 128;    // bytes of a 64 x 64 tile of 16-bit operands
constexpr uint32_t STAGE = 4 * BOX;   // a CTA's halves: A 128 x 64, B 128 x 64
constexpr uint32_t STG = 32 * 128;    // a warp's staging tile: 32 rows of 128 bytes
constexpr size_t SMEM_BAR = 512;
constexpr uint64_t WAIT_NS = 2000000000ull;

constexpr int stages(int mode) { return mode == kCeLse ? 7 : 5; }
constexpr size_t smem_bytes(int mode) {
  return 1024 + (size_t)stages(mode) * STAGE + (mode == kCeLse ? 0 : EPI_WARPS * STG) + SMEM_BAR;
}
static_assert(smem_bytes(kCeLse) <= 232448 && smem_bytes(kCeGrad) <= 232448, "above the per-block limit");

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

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void tma_add_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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

// 64-row boxes of the A operand that a CTA loads in the score modes: with one
// tile of rows, those that hold rows. The others are zeroed once.
__device__ __forceinline__ int a_boxes(const CeGemm& a, int cta) {
  return a.one_tile_rows ? max(0, min(2, (a.one_tile_rows - cta * 128 + 63) / 64)) : 2;
}

struct Tiles {
  int mtiles;         // rows that take part, in tiles
  int kblocks_rows;   // and in K blocks
  int n_dx, n_dw;
  int total;
};

template <int MODE>
__device__ __forceinline__ Tiles count_tiles(const CeGemm& a) {
  Tiles t;
  const int rows = taken_rows(a);
  t.mtiles = (rows + kCeM - 1) / kCeM;
  t.kblocks_rows = (rows + kCeK - 1) / kCeK;
  t.n_dx = t.n_dw = 0;
  if (MODE == kCeStore) {
    if (a.dx.on) t.n_dx = t.mtiles * a.dx.ntiles * a.dx.splits;
    if (a.dw.on) t.n_dw = a.dw.mtiles * a.dw.ntiles * a.dw.splits;
    t.total = t.n_dx + t.n_dw;
  } else {
    t.total = t.mtiles * a.vtiles;
  }
  return t;
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
  // The longer product's tiles first, so the shorter ones fill the last turn.
  const int n_first = a.dw_first ? c.n_dw : c.n_dx;
  const bool second = id >= n_first;
  t.job = (a.dw_first != 0) != second;
  if (second) id -= n_first;
  const CeJob& j = t.job ? a.dw : a.dx;
  t.n = id % j.ntiles * kCeN;
  id /= j.ntiles;
  t.split = id % j.splits;
  t.m = id / j.splits;
  t.bn = a.d - t.n > 128 ? 256 : 128;
  const int kb = t.job ? c.kblocks_rows : j.kblocks;
  const int per = (kb + j.splits - 1) / j.splits;
  t.kb0 = min(kb, t.split * per);
  t.kb1 = min(kb, t.kb0 + per);
  return t;
}

// --------------------------------------------------------------- epilogues

// 64 scores of a row: their maximum and the sum of powers of two (the scores
// times scale * log2(e), so that e^z is one ex2), and the target's score.
__device__ __forceinline__ void epi_lse(const CeGemm& a, float (&w)[QCOLS], int n0, int64_t row, bool live, int tgt) {
  const int cols = a.classes - n0;
  if (cols <= 0) return;
  if (cols < QCOLS) {
#pragma unroll
    for (int j = 0; j < QCOLS; j++)
      if (j >= cols) w[j] = -INFINITY;
  }
  const int at = tgt - n0;
  if (at >= 0 && at < QCOLS && live) {
    float z = 0.0f;
#pragma unroll
    for (int j = 0; j < QCOLS; j++) z = j == at ? w[j] : z;
    a.zt[row] = z * a.c2;
  }
  float m[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    m[k] = fmax3(w[16 * k], w[16 * k + 1], w[16 * k + 2]);
#pragma unroll
    for (int j = 3; j < 15; j += 2) m[k] = fmax3(m[k], w[16 * k + j], w[16 * k + j + 1]);
    m[k] = fmaxf(m[k], w[16 * k + 15]);
  }
  const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * a.c2;
  const float sub = top == -INFINITY ? 0.0f : top;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < QCOLS; j++) sum[j & 3] += ex2(fmaf(w[j], a.c2, -sub));
  if (live) a.part[row * a.parts + n0 / QCOLS] = make_float2(top, (sum[0] + sum[1]) + (sum[2] + sum[3]));
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

// 64 values of a row in 16 bits into the staging tile.
template <bool F16>
__device__ __forceinline__ void stage_row16(uint8_t* stg, int lane, const float (&w)[QCOLS]) {
#pragma unroll
  for (int q = 0; q < 8; q++)
    stage_put(stg, lane, q,
              make_uint4(pack2<F16>(w[8 * q], w[8 * q + 1]), pack2<F16>(w[8 * q + 2], w[8 * q + 3]),
                         pack2<F16>(w[8 * q + 4], w[8 * q + 5]), pack2<F16>(w[8 * q + 6], w[8 * q + 7])));
}

// ------------------------------------------------------------------ kernel

template <int MODE, bool F16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    ce_gemm_kernel(const __grid_constant__ CeMaps maps, const __grid_constant__ CeGemm a) {
  constexpr int ST = stages(MODE);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_stg = smem + (size_t)ST * STAGE;
  uint64_t* bars = (uint64_t*)(s_stg + (MODE == kCeLse ? 0 : EPI_WARPS * STG));
  uint64_t* full = bars;           // [ST] even CTA: both CTAs' bytes
  uint64_t* empty = full + ST;     // [ST] each CTA: MMA commit
  uint64_t* tfull = empty + ST;    // [2] each CTA: MMA commit
  uint64_t* tempty = tfull + 2;    // [2] even CTA: both CTAs' epilogue warps
  uint32_t* s_tmem = (uint32_t*)(tempty + 2);
  volatile int* s_abort = (volatile int*)(s_tmem + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = (int)cluster_ctarank();
  const bool lead = cta == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * EPI_WARPS);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc_pair(s_tmem, 512);
  if (MODE != kCeStore && a.one_tile_rows) {
    const int skip = a_boxes(a, cta) * (int)BOX;
    for (int s = 0; s < ST; s++)
      for (int i = skip + threadIdx.x * 16; i < 2 * (int)BOX; i += THREADS * 16)
        *reinterpret_cast<uint4*>(smem + s * STAGE + i) = make_uint4(0, 0, 0, 0);
    fence_async_smem();
  }
  tc_fence_before();
  cluster_sync();  // barriers initialised and TMEM allocated in both CTAs
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // The set-up above overlaps the end of the kernel before; its results are
  // there from here on.
  grid_launch();
  grid_wait();
  const Tiles cnt = count_tiles<MODE>(a);

  if (warp == 0) {
    // ---------------------------------------------------- TMA producer
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      const int na = a_boxes(a, cta);
      for (int id = pair; ok && id < cnt.total; id += npairs) {
        const Tile t = tile_at<MODE>(a, cnt, id);
        const int boxes = t.bn >> 7;  // of B in each CTA
        const uint32_t bytes = (MODE == kCeStore ? 4 : a_boxes(a, 0) + a_boxes(a, 1)) * BOX + 2u * boxes * BOX;
        const int ra = t.m * kCeM + cta * 128;
        const int rb = t.n + cta * (t.bn >> 1);
        for (int kb = t.kb0; kb < t.kb1; kb++, it++) {
          const int s = it % ST;
          if (!mbar_wait(&empty[s], ((it / ST) & 1) ^ 1, s_abort, a.err, 31, WAIT_NS)) {
            ok = false;
            break;
          }
          if (lead) mbar_expect_tx(&full[s], bytes);
          const uint32_t bar = mapa_shared(&full[s], 0);
          uint8_t* sa = smem + s * STAGE;
          uint8_t* sb = sa + 2 * BOX;
          const int k = kb * kCeK;
          if (MODE != kCeStore) {
            for (int i = 0; i < na; i++) tma_load_2d_pair(sa + i * BOX, &maps.x, k, ra + 64 * i, bar);
            for (int i = 0; i < boxes; i++) tma_load_2d_pair(sb + i * BOX, &maps.w, k, a.v0 + rb + 64 * i, bar);
          } else if (t.job == 0) {
            for (int i = 0; i < 2; i++) tma_load_2d_pair(sa + i * BOX, &maps.g, k, ra + 64 * i, bar);
            for (int i = 0; i < boxes; i++) tma_load_2d_pair(sb + i * BOX, &maps.w, rb + 64 * i, a.v0 + k, bar);
          } else {
            for (int i = 0; i < 2; i++) tma_load_2d_pair(sa + i * BOX, &maps.g, ra + 64 * i, k, bar);
            for (int i = 0; i < boxes; i++) tma_load_2d_pair(sb + i * BOX, &maps.x, rb + 64 * i, k, bar);
          }
        }
      }
      if (*s_abort && lead) {
        // Drain (bounded): both CTAs' loads complete on these barriers.
        volatile int dummy = 0;
        for (int i = max(0, it - ST); i < it; i++)
          mbar_wait(&full[i % ST], (i / ST) & 1, &dummy, a.err, 0, WAIT_NS / 4);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------- MMA issuer (even CTA)
    if (lane == 0 && lead) {
      int it = 0, tn = 0, last = -1;
      bool ok = true;
      for (int id = pair; ok && id < cnt.total; id += npairs, tn++) {
        const Tile t = tile_at<MODE>(a, cnt, id);
        const int b = tn & 1;
        if (!mbar_wait(&tempty[b], ((tn >> 1) & 1) ^ 1, s_abort, a.err, 32, WAIT_NS)) break;
        tc_fence_after();
        // (A split without K blocks commits at once: its epilogue stores zeros.)
        const uint32_t d = tmem + b * 256;
        const bool a_mn = MODE == kCeStore && t.job == 1, b_mn = MODE == kCeStore;
        const uint32_t idesc = a.idesc | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(t.bn >> 3) << 17);
        for (int kb = t.kb0; kb < t.kb1; kb++, it++) {
          const int s = it % ST;
          if (!mbar_wait(&full[s], (it / ST) & 1, s_abort, a.err, 33, WAIT_NS)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint8_t* sa = smem + s * STAGE;
          const uint64_t ad = a_mn ? desc_mn(sa) : smem_desc_sw128(sa);
          const uint64_t bd = b_mn ? desc_mn(sa + 2 * BOX) : smem_desc_sw128(sa + 2 * BOX);
          // 16 of K: 32 bytes on in a K-major row, 16 rows on in an MN-major
          // box. (Shared addresses are below 2^18: no carry out of the field.)
          const uint32_t astep = a_mn ? 2048 >> 4 : 32 >> 4, bstep = b_mn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
          for (int ks = 0; ks < 4; ks++)
            mma_f16_pair(d, ad + ks * astep, bd + ks * bstep, idesc, kb > t.kb0 || ks > 0 ? 1u : 0u);
          mma_commit_pair(&empty[s], 0x3);
        }
        mma_commit_pair(&tfull[b], 0x3);
        last = tn;
      }
      if (*s_abort && last >= 0) {
        volatile int dummy = 0;
        mbar_wait(&tfull[last & 1], (last >> 1) & 1, &dummy, a.err, 0, WAIT_NS / 4);
      }
    }
  } else if (warp >= EPI_FIRST) {
    // ---------------------------------------------------- epilogue
    const int quarter = (warp - EPI_FIRST) >> 2, quad = warp & 3;
    uint8_t* stg = s_stg + (warp - EPI_FIRST) * STG;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int taken = taken_rows(a);
    int tn = 0;
    for (int id = pair; id < cnt.total; id += npairs, tn++) {
      const Tile t = tile_at<MODE>(a, cnt, id);
      const int b = tn & 1;
      const int r0 = t.m * kCeM + cta * 128 + quad * 32;  // the warp's first row
      const int64_t row = r0 + lane;
      const int n0 = t.n + quarter * QCOLS;               // and column
      const bool mine = quarter * QCOLS < t.bn && (MODE != kCeLse || r0 < taken);
      const bool live = row < taken;
      int tgt = -1;
      float lse2 = 0.0f, gs = 0.0f;
      if (MODE != kCeStore && live) {
        if (a.targets) {  // unpacked rows
          const int64_t g = a.targets[row];
          tgt = g >= 0 && g < a.classes ? (int)g : -1;
        } else {
          tgt = a.target[row];
        }
        if (MODE == kCeGrad) {
          lse2 = a.lse2[row];
          gs = a.gs[row];
        }
      }
      const bool ok = mbar_wait(&tfull[b], (tn >> 1) & 1, s_abort, a.err, 34, WAIT_NS);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      float w[QCOLS];
      if (mine) tmem_ld64(tmem + lanes + b * 256 + quarter * QCOLS, w);
      // The columns are in registers: hand the accumulator back.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (lead)
          mbar_arrive(&tempty[b]);
        else
          mbar_arrive_cluster(mapa_shared(&tempty[b], 0));
      }
      if (!mine) continue;
      if (MODE == kCeLse) {
        epi_lse(a, w, n0, row, live, tgt);
      } else if (MODE == kCeGrad) {
        // g = (2^(c2 z - lse2) - [target]) gs in 16 bits; zeros past the last
        // class and in the tail rows, which the products read.
        const int cols = a.vn - n0;
#pragma unroll
        for (int j = 0; j < QCOLS; j++) w[j] = ex2(fmaf(w[j], a.c2, -lse2));
        const int at = tgt - a.v0 - n0;
        if (at >= 0 && at < QCOLS) {
#pragma unroll
          for (int j = 0; j < QCOLS; j++)
            if (j == at) w[j] -= 1.0f;
        }
#pragma unroll
        for (int j = 0; j < QCOLS; j++) w[j] *= gs;
        if (cols < QCOLS || !live) {
#pragma unroll
          for (int j = 0; j < QCOLS; j++)
            if (!live || j >= cols) w[j] = 0.0f;
        }
        stage_ready(lane);
        stage_row16<F16>(stg, lane, w);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&maps.g_out, stg, n0, r0);
          bulk_commit();
        }
      } else {
        const CeJob& j = t.job ? a.dw : a.dx;
        const CUtensorMap* out = t.job ? &maps.dw_out : &maps.dx_out;
        if (n0 >= a.d) continue;  // past the last column
        if (t.kb0 == t.kb1) {
#pragma unroll
          for (int i = 0; i < QCOLS; i++) w[i] = 0.0f;
        }
        if (j.f32_rows > 0) {
          // whole tiles of rows: never past the end of the split's result
          const int y = t.split * j.f32_rows + r0;
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (n0 + h * 32 >= a.d) break;
            stage_ready(lane);
#pragma unroll
            for (int q = 0; q < 8; q++)
              stage_put(stg, lane, q,
                        make_uint4(__float_as_uint(w[32 * h + 4 * q]), __float_as_uint(w[32 * h + 4 * q + 1]),
                                   __float_as_uint(w[32 * h + 4 * q + 2]), __float_as_uint(w[32 * h + 4 * q + 3])));
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (j.add)
                tma_add_2d(out, stg, n0 + h * 32, y);
              else
                tma_store_2d(out, stg, n0 + h * 32, y);
              bulk_commit();
            }
          }
        } else {
          const float f = a.head->grad_scale;
#pragma unroll
          for (int i = 0; i < QCOLS; i++) w[i] *= f;
          stage_ready(lane);
          stage_row16<F16>(stg, lane, w);
          fence_async_smem();
          __syncwarp();
          if (!j.out) {
            if (lane == 0) {
              tma_store_2d(out, stg, n0, j.row0 + r0);
              bulk_commit();
            }
          } else {
            // Rows that TMA cannot address: the warp stores them one by one,
            // two elements a lane.
            const int64_t left = a.classes - (j.row0 + (int64_t)r0);
            uint16_t* o = j.out + (j.row0 + (int64_t)r0) * j.out_stride + n0;
            const int cols = a.d - n0;
            for (int r = 0; r < 32 && r < left; r++, o += j.out_stride) {
#pragma unroll
              for (int h = 0; h < 2; h++) {
                const int c = lane + 32 * h;
                if (c < cols) o[c] = *reinterpret_cast<uint16_t*>(stg + r * 128 + ((((c >> 3) ^ (r & 7)) << 4) | (c & 7) << 1));
              }
            }
            __syncwarp();
          }
        }
      }
    }
    if (MODE != kCeLse && lane == 0) bulk_wait_all();  // shared memory is read until then
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no MMA, load or remote arrival of either CTA is still pending
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Pairs of the kernel that the current device runs at the same time, asked
// once per device (with the shared memory that the kernel needs allowed).
template <int MODE, bool F16>
int pairs_of(int* out) {
  static std::atomic<int> cached[128];
  int dev = 0;
  VRS_CUDA(cudaGetDevice(&dev));
  int n = dev < 128 ? cached[dev].load() : 0;
  if (n == 0) {
    auto kernel = ce_gemm_kernel<MODE, F16>;
    VRS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(MODE)));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem_bytes(MODE);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    VRS_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    if (n < 1) {
      set_error(VRS_ERR_DRIVER, "linear cross entropy: no CTA pair of the product kernel fits this device");
      return VRS_ERR_DRIVER;
    }
    if (dev < 128) cached[dev].store(n);
  }
  *out = n;
  return VRS_OK;
}

template <int MODE, bool F16>
int launch(const CeMaps& maps, const CeGemm& a, int64_t most_tiles, cudaStream_t s) {
  int pairs = 0;
  VRS_TRY((pairs_of<MODE, F16>(&pairs)));
  const int64_t n = most_tiles < pairs ? most_tiles : pairs;
  VRS_TRY(launch_after(ce_gemm_kernel<MODE, F16>, (unsigned)(2 * (n < 1 ? 1 : n)), THREADS, smem_bytes(MODE), s, maps, a));
  count_launch();
  return VRS_OK;
}

}  // namespace

int launch_ce_gemm(int mode, bool is_f16, const CeMaps& maps, const CeGemm& a, int64_t most_tiles, cudaStream_t s) {
  switch (mode) {
    case kCeLse: return is_f16 ? launch<kCeLse, true>(maps, a, most_tiles, s) : launch<kCeLse, false>(maps, a, most_tiles, s);
    case kCeGrad: return is_f16 ? launch<kCeGrad, true>(maps, a, most_tiles, s) : launch<kCeGrad, false>(maps, a, most_tiles, s);
    default: return is_f16 ? launch<kCeStore, true>(maps, a, most_tiles, s) : launch<kCeStore, false>(maps, a, most_tiles, s);
  }
}

}  // namespace ops
}  // namespace vrs
