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
// accumulators (2 x 256 columns = all of TMEM); two groups of four epilogue
// warps a CTA take alternate tiles, so a tile is drained, exponentiated and
// stored while the next one is multiplied. Results leave through swizzled
// staging tiles and TMA stores, in f32 also as TMA additions to what earlier
// pieces of the classes left.
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

constexpr int THREADS = 384;          // producer, MMA, TMEM, spare; 8 epilogue warps
constexpr int EPI_FIRST = 4;
constexpr uint32_t BOX = 64 * 128;    // bytes of a 64 x 64 tile of 16-bit operands
constexpr uint32_t STAGE = 4 * BOX;   // a CTA's halves: A 128 x 64, B 128 x 64
constexpr uint32_t STG = 32 * 128;    // a warp's staging tile: 32 rows of 128 bytes
constexpr size_t SMEM_BAR = 512;
constexpr uint64_t WAIT_NS = 2000000000ull;

constexpr int stages(int mode) { return mode == kCeLse ? 6 : 5; }
constexpr size_t smem_bytes(int mode) {
  return 1024 + (size_t)stages(mode) * STAGE + (mode == kCeLse ? 0 : 8 * 2 * STG) + SMEM_BAR;
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

// 32 lanes x 32 columns; the values may be used only after tmem_wait.
__device__ __forceinline__ void tmem_ld_issue(uint32_t taddr, float (&v)[32]) {
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
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
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

struct Tiles {
  int mtiles;         // rows that take part, in tiles
  int kblocks_rows;   // and in K blocks
  int n_dx, n_dw;
  int total;
};

template <int MODE>
__device__ __forceinline__ Tiles count_tiles(const CeGemm& a) {
  Tiles t;
  const int rows = a.head->taken;
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
    t.n = id / c.mtiles * kCeN;
    t.bn = kCeN;
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

// One row's 256 scores: running maximum and sum of powers of two (the scores
// times scale * log2(e), so that e^z is one ex2), the target's score.
__device__ __forceinline__ void epi_lse(const CeGemm& a, uint32_t tmem, int n0, int64_t row, bool live, int tgt,
                                        int vtile) {
  float top = -INFINITY, sum = 0.0f;
  const int cols = min(kCeN, a.classes - n0);
  float v[2][32];
  tmem_ld_issue(tmem, v[0]);
#pragma unroll
  for (int c = 0; c < kCeN / 32; c++) {
    float(&w)[32] = v[c & 1];
    tmem_wait(w);
    if (c + 1 < kCeN / 32) tmem_ld_issue(tmem + (c + 1) * 32, v[(c + 1) & 1]);
    if (c * 32 >= cols) continue;
    if (cols - c * 32 < 32) {
#pragma unroll
      for (int j = 0; j < 32; j++)
        if (j >= cols - c * 32) w[j] = -INFINITY;
    }
    const int at = tgt - n0 - c * 32;
    if (at >= 0 && at < 32) {
      float z = 0.0f;
#pragma unroll
      for (int j = 0; j < 32; j++) z = j == at ? w[j] : z;
      if (live) a.zt[row] = z * a.c2;
    }
    float m = fmaxf(w[0], w[1]);
#pragma unroll
    for (int j = 2; j < 32; j += 2) m = fmax3(m, w[j], w[j + 1]);
    m *= a.c2;
    if (m > top) {
      sum *= ex2(top - m);
      top = m;
    }
    const float sub = top == -INFINITY ? 0.0f : top;
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      s0 += ex2(fmaf(w[j], a.c2, -sub));
      s1 += ex2(fmaf(w[j + 1], a.c2, -sub));
    }
    sum += s0 + s1;
  }
  if (live) a.part[row * a.vtiles + vtile] = make_float2(top, sum);
}

// A staging tile is free again once its last store has read it (of two).
__device__ __forceinline__ void stage_ready(int lane) {
  if (lane == 0) bulk_wait_read<1>();
  __syncwarp();
}

// Row `lane` of a staging tile: 16-byte chunk j, 128-byte swizzle.
__device__ __forceinline__ void stage_put(uint8_t* stg, int lane, int j, uint4 q) {
  *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = q;
}

// ------------------------------------------------------------------ kernel

template <int MODE, bool F16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    ce_gemm_kernel(const __grid_constant__ CeMaps maps, const __grid_constant__ CeGemm a) {
  constexpr int ST = stages(MODE);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_stg = smem + (size_t)ST * STAGE;
  uint64_t* bars = (uint64_t*)(s_stg + (MODE == kCeLse ? 0 : 8 * 2 * STG));
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
      mbar_init(&tempty[b], 8);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc_pair(s_tmem, 512);
  tc_fence_before();
  cluster_sync();  // barriers initialised and TMEM allocated in both CTAs
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const Tiles cnt = count_tiles<MODE>(a);

  if (warp == 0) {
    // ---------------------------------------------------- TMA producer
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int id = pair; ok && id < cnt.total; id += npairs) {
        const Tile t = tile_at<MODE>(a, cnt, id);
        const int boxes = t.bn >> 7;  // of B in each CTA
        const int ra = t.m * kCeM + cta * 128;
        const int rb = t.n + cta * (t.bn >> 1);
        for (int kb = t.kb0; kb < t.kb1; kb++, it++) {
          const int s = it % ST;
          if (!mbar_wait(&empty[s], ((it / ST) & 1) ^ 1, s_abort, a.err, 31, WAIT_NS)) {
            ok = false;
            break;
          }
          if (lead) mbar_expect_tx(&full[s], 2u * (2 + boxes) * BOX);
          const uint32_t bar = mapa_shared(&full[s], 0);
          uint8_t* sa = smem + s * STAGE;
          uint8_t* sb = sa + 2 * BOX;
          const int k = kb * kCeK;
          if (MODE != kCeStore) {
            for (int i = 0; i < 2; i++) tma_load_2d_pair(sa + i * BOX, &maps.x, k, ra + 64 * i, bar);
            for (int i = 0; i < 2; i++) tma_load_2d_pair(sb + i * BOX, &maps.w, k, a.v0 + rb + 64 * i, bar);
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
    const int group = (warp - EPI_FIRST) >> 2, quad = warp & 3;
    uint8_t* stg = s_stg + (warp - EPI_FIRST) * 2 * STG;
    int puts = 0;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + group * 256;
    int tn = 0;
    for (int id = pair; id < cnt.total; id += npairs, tn++) {
      if ((tn & 1) != group) continue;
      const Tile t = tile_at<MODE>(a, cnt, id);
      const int r0 = t.m * kCeM + cta * 128 + quad * 32;  // the warp's first row
      const int64_t row = r0 + lane;
      int tgt = -1;
      float lse2 = 0.0f, gs = 0.0f;
      const bool any = MODE == kCeStore ? true : r0 < a.head->taken;
      const bool live = row < a.head->taken;
      if (MODE != kCeStore && live) {
        tgt = a.target[row];
        if (MODE == kCeGrad) {
          lse2 = a.lse2[row];
          gs = a.gs[row];
        }
      }
      const bool ok = mbar_wait(&tfull[group], (tn >> 1) & 1, s_abort, a.err, 34, WAIT_NS);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      if (MODE == kCeLse) {
        if (any) epi_lse(a, taddr, t.n, row, live, tgt, t.n / kCeN);
      } else if (MODE == kCeGrad) {
        // g = (2^(c2 z - lse2) - [target]) gs in 16 bits; zeros past the last
        // class and in the tail rows, which the products read.
        const int cols = min(kCeN, a.vn - t.n);
        tgt -= a.v0 + t.n;
        float v[2][32];
        if (any) tmem_ld_issue(taddr, v[0]);
#pragma unroll
        for (int c = 0; c < kCeN / 32; c++) {
          float(&w)[32] = v[c & 1];
          if (any) {
            tmem_wait(w);
            if (c + 1 < kCeN / 32) tmem_ld_issue(taddr + (c + 1) * 32, v[(c + 1) & 1]);
#pragma unroll
            for (int j = 0; j < 32; j++) w[j] = ex2(fmaf(w[j], a.c2, -lse2));
            const int at = tgt - c * 32;
            if (at >= 0 && at < 32) {
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (j == at) w[j] -= 1.0f;
            }
#pragma unroll
            for (int j = 0; j < 32; j++) w[j] *= gs;
            if (!live) {
#pragma unroll
              for (int j = 0; j < 32; j++) w[j] = 0.0f;
            }
            if (cols - c * 32 < 32) {
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (j >= cols - c * 32) w[j] = 0.0f;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j++) w[j] = 0.0f;
          }
          uint8_t* to = stg + (puts & 1) * STG;
          if ((c & 1) == 0) stage_ready(lane);
#pragma unroll
          for (int q = 0; q < 4; q++)
            stage_put(to, lane, (c & 1) * 4 + q,
                      make_uint4(pack2<F16>(w[8 * q], w[8 * q + 1]), pack2<F16>(w[8 * q + 2], w[8 * q + 3]),
                                 pack2<F16>(w[8 * q + 4], w[8 * q + 5]), pack2<F16>(w[8 * q + 6], w[8 * q + 7])));
          if (c & 1) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&maps.g_out, to, t.n + (c - 1) * 32, r0);
              bulk_commit();
            }
            puts++;
          }
        }
      } else {
        const CeJob& j = t.job ? a.dw : a.dx;
        const bool none = t.kb0 == t.kb1;
        const bool f32 = j.f32_rows > 0;
        const CUtensorMap* out = t.job ? &maps.dw_out : &maps.dx_out;
        // rows of the f32 result are never past its end: whole tiles
        const int y = f32 ? t.split * j.f32_rows + r0 : j.row0 + r0;
        const float f = a.head->grad_scale;
        for (int c = 0; c < t.bn / 32; c++) {
          float w[32];
          if (none) {
#pragma unroll
            for (int i = 0; i < 32; i++) w[i] = 0.0f;
          } else {
            tmem_ld_issue(taddr + c * 32, w);
            tmem_wait(w);
          }
          if (t.n + c * 32 >= a.d) {
            if (f32 || (c & 1) == 0) break;  // past the last column; a 16-bit tile half written still goes out
          }
          uint8_t* to = stg + (puts & 1) * STG;
          if (f32) {
            stage_ready(lane);
#pragma unroll
            for (int q = 0; q < 8; q++)
              stage_put(to, lane, q,
                        make_uint4(__float_as_uint(w[4 * q]), __float_as_uint(w[4 * q + 1]),
                                   __float_as_uint(w[4 * q + 2]), __float_as_uint(w[4 * q + 3])));
          } else {
            if ((c & 1) == 0) stage_ready(lane);
#pragma unroll
            for (int i = 0; i < 32; i++) w[i] *= f;
#pragma unroll
            for (int q = 0; q < 4; q++)
              stage_put(to, lane, (c & 1) * 4 + q,
                        make_uint4(pack2<F16>(w[8 * q], w[8 * q + 1]), pack2<F16>(w[8 * q + 2], w[8 * q + 3]),
                                   pack2<F16>(w[8 * q + 4], w[8 * q + 5]), pack2<F16>(w[8 * q + 6], w[8 * q + 7])));
          }
          if (f32 || (c & 1)) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (!f32)
                tma_store_2d(out, to, t.n + (c - 1) * 32, y);
              else if (j.add)
                tma_add_2d(out, to, t.n + c * 32, y);
              else
                tma_store_2d(out, to, t.n + c * 32, y);
              bulk_commit();
            }
            puts++;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (lead)
          mbar_arrive(&tempty[group]);
        else
          mbar_arrive_cluster(mapa_shared(&tempty[group], 0));
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
  ce_gemm_kernel<MODE, F16><<<(unsigned)(2 * (n < 1 ? 1 : n)), THREADS, smem_bytes(MODE), s>>>(maps, a);
  VRS_CUDA(cudaGetLastError());
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
