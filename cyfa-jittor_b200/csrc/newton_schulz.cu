// Newton-Schulz orthogonalisation of a batch of matrices G [m, n] (the update of
// the Muon optimiser): with X0 = G / (|G|_F + eps), taken as [M, N], M <= N
// (transposed when G is tall),
//   A = X X^T,   B = b A + c A A,   X <- a X + B X        (each step)
// which pushes every singular value towards 1.
//
// The products run on tcgen05 (CTA pairs) with fp32 accumulators in TMEM.  X, A
// and B are kept as fp16 pairs hi + lo (22 significant bits), stored times 2^12:
// that keeps the lo parts of small entries above fp16's underflow and leaves room
// up to |entry| < 16.  Every product is the three MMAs hi hi + hi lo + lo hi: lo lo is
// 2^-22 of it.  (hi hi alone, in X X^T and in the first steps, where fewer terms cancel,
// took 2.5 ms in place of 3.5 for 24 matrices of 2816 x 1024, but left 6e-4 after five
// steps, a third of the result's rounding, and more than that rounding after 16: the
// quintic's fixed value repels, so that long runs enlarge what is lost.)
// A and B are symmetric: only the tiles on and below the diagonal are computed,
// the others are written as their mirror images.
//
// Bound by the tensor cores' rate: of five steps on 24 bf16 matrices of 2816 x 1024
// (3.5 ms in all), B X takes 300 us a step (425 GFLOP as issued, 1.42 PFLOP/s), X X^T 219
// (266 GFLOP, 1.22: its 240 tiles are four rounds of 74 CTA pairs, the last a quarter
// full), b A + c A A 92; splitting G into X0 100 and its norms 31.  Four matrices of
// 127 x 509 take 116 us: 15 products one after the other.
#include <cuda_fp16.h>

#include "cyfa_common.cuh"

namespace cyfa {

constexpr float kNsScale = 4096.f;  // 2^12
constexpr int kNsEpi = 8;            // finishing warps
constexpr int kNsThreads = (kNsEpi + 2) * 32;
constexpr int kNsTile = 256;  // rows and columns of a CTA pair's tile
// Matrices of up to 128 rows: one CTA takes all steps of a matrix in one launch, if
// they are short, low or many enough; otherwise their columns' tiles are spread over the
// SMs at three launches a step (five steps, f32, with the norms and X0, in us; one CTA a
// matrix against spread: 4 of 128 x 512 112 and 152, of 1024 164 and 185, 1 of 2048 268 and
// 252, 4 of 4096 472 and 390; 32 of 4096 607 and 581, 48 of 2048 339 and 413, 64 of 4096
// 668 and 820; 4 of 32 x 8192 565 and 639).
constexpr int kNsSoloWidth = 1024, kNsSoloCount = 48, kNsSoloRows = 32;

enum NsMode : int {
  kNsGram = 0,    // D = acc
  kNsPoly = 1,    // D = alpha acc + beta C
  kNsStep = 2,    // D = acc + beta C, row-major
  kNsLast = 3,    // the step's result as bf16, in G's orientation
};

struct NsGemmParams {
  int L, M, cols, K;        // D [L, M, cols] = contraction over K
  int tiles_m;
  int nunits, per;          // tiles in all, tiles of one matrix
  float alpha, beta;
  __nv_bfloat16* out;       // kNsLast
  int tall;                 // out is [L, cols, M]
  float diag;               // and a in the units of D, added to B's diagonal
};

// Per stage and CTA: 128 rows of A and 128 of B, 64 contraction columns each, hi and lo.
constexpr int kNsPart = 128 * 128;
constexpr int kNsSlot = 32 * 64;  // a finishing warp's block: 32 rows x 32 columns of 16 bits
constexpr int kNsStageBytes = 4 * kNsPart, kNsStages = 3;
constexpr int kNsSmem = kNsStages * kNsStageBytes + kNsEpi * 2 * kNsSlot + 1024;

// fp16 x fp16 -> fp32
__host__ __device__ constexpr uint32_t ns_idesc(int M, int N, int b_mn) {
  return (1u << 4) | (uint32_t(b_mn) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

// Unit u -> (matrix, row tile, column tile).  Symmetric products skip the tiles
// above the diagonal: row tile i has the column tiles 0 .. i.
struct NsTile {
  int l, ti, tj;
};
template <bool SYM>
__device__ __forceinline__ NsTile ns_tile(const NsGemmParams& p, int u) {
  NsTile t;
  t.l = u / p.per;
  int r = u - t.l * p.per;
  if (SYM) {
    t.ti = 0;
    while (r > t.ti) {
      ++t.ti;
      r -= t.ti;
    }
    t.tj = r;
  } else {
    t.ti = r % p.tiles_m;
    t.tj = r / p.tiles_m;
  }
  return t;
}

// ------------------------------------------------ finishing a tile
// A finishing warp's blocks of 32 x 32 16-bit entries in shared memory, laid out as
// the 64-byte TMA swizzle: 4 chunks of 16 bytes a row.  A lane reads and writes its
// own row; memory is reached by TMA.  (Going to memory from the registers, by rows
// or through a warp transposition, cost more load/store issue than the tile's
// MMAs take: 209 us against 140 for B X with one MMA a product, on 24 matrices of 1024 x 2816.)
__device__ __forceinline__ uint32_t ns_slot(uint32_t block, int row, int chunk) {
  return block + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
// v += beta * the block's row `lane`
__device__ __forceinline__ void ns_add(uint32_t block, float beta, float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 u = ld_shared_v4(ns_slot(block, lane, c));
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = __half22float2(h[e]);
      v[8 * c + 2 * e] = fmaf(beta, x.x, v[8 * c + 2 * e]);
      v[8 * c + 2 * e + 1] = fmaf(beta, x.y, v[8 * c + 2 * e + 1]);
    }
  }
}
// row: the lane's 32 entries, two to a word
__device__ __forceinline__ void ns_put(uint32_t block, const uint32_t (&row)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    st_shared_v4(ns_slot(block, lane, c), row[4 * c], row[4 * c + 1], row[4 * c + 2],
                 row[4 * c + 3]);
}
// The block transposed: 8 x 8 pieces read with their transposition into t, then
// written back as the pieces of the transposed block.
__device__ __forceinline__ void ns_read_transposed(uint32_t block, uint32_t (&t)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(t[4 * g]), "=r"(t[4 * g + 1]), "=r"(t[4 * g + 2]), "=r"(t[4 * g + 3])
                 : "r"(ns_slot(block, lane, g))
                 : "memory");
}
__device__ __forceinline__ void ns_write_transposed(uint32_t block, const uint32_t (&t)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                     ns_slot(block, 8 * g + (lane & 7), lane >> 3)),
                 "r"(t[4 * g]), "r"(t[4 * g + 1]), "r"(t[4 * g + 2]), "r"(t[4 * g + 3])
                 : "memory");
}
// The block to rows of dst (stride ld), 8 rows x 64 bytes at a time or, for rows at
// any alignment, one row at a time; rows from `rows` and columns from `cols` on are
// left out.
__device__ __forceinline__ void ns_store(uint32_t block, __nv_bfloat16* dst, long long ld, int rows,
                                         int cols, bool aligned16) {
  const int lane = threadIdx.x & 31;
  if (aligned16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = 8 * k + (lane >> 2), c = lane & 3;
      const uint4 u = ld_shared_v4(ns_slot(block, r, c));
      if (r < rows && c * 8 < cols) *reinterpret_cast<uint4*>(dst + r * ld + c * 8) = u;
    }
  } else {
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      uint16_t u;
      asm volatile("ld.shared.u16 %0, [%1];"
                   : "=h"(u)
                   : "r"(ns_slot(block, r, lane >> 3) + (lane & 7) * 2));
      if (r < rows && lane < cols) dst[r * ld + lane] = __ushort_as_bfloat16(u);
    }
  }
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// hi parts of v packed into w, v becomes what they leave
__device__ __forceinline__ void ns_split_row(float (&v)[32], uint32_t (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    w[e] = pack_half2(v[2 * e], v[2 * e + 1]);
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
    v[2 * e] -= h.x;
    v[2 * e + 1] -= h.y;
  }
}

// ------------------------------------------------ CTA pair (cta_group::2)
// Tile load into this CTA's shared memory, completion signalled on the barrier
// at the cluster address `bar` (the leader's).
// The load and MMA warps run converged, all addresses warp-uniform, and one lane issues:
// with a single lane inside a divergent branch each operand was moved to the uniform
// registers for every instruction, 1400 cycles for a 64-column block whose MMAs take
// 1536, and 500 cycles for a load.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e;
}
template <bool PAIR>
__device__ __forceinline__ void ns_load(uint32_t lane_on, void* dst, const void* tmap, uint32_t bar, int x,
                                        int y, int z) {
  if (PAIR)
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"
        " @q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];\n}\n" ::"r"(smem_u32(dst)),
        "l"(tmap), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(lane_on)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"
        " @q cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];\n}\n" ::"r"(smem_u32(dst)),
        "l"(tmap), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(lane_on)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void ns_umma(uint32_t lane_on, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lane_on));
  else
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lane_on));
}
// Arrives on the barrier (PAIR: at this address in both CTAs) when the MMAs issued so
// far are done.
template <bool PAIR>
__device__ __forceinline__ void ns_commit(uint32_t lane_on, uint64_t* bar) {
  if (PAIR)
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
        " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;\n}\n" ::"r"(smem_u32(bar)),
        "h"(static_cast<uint16_t>(3)), "r"(lane_on)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
            smem_u32(bar)),
        "r"(lane_on)
        : "memory");
}
__device__ __forceinline__ void cluster_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// TMA addresses of the finishing warps: C and D as pairs of 32 x 32 blocks.
struct NsEpiMaps {
  CUtensorMap ch, cl, dh, dl;
};

// Persistent CTA pairs; a pair's tile is 256 x 256, CTA r of it holds rows 128 r ..
// of the result (in its TMEM) and of A, and columns 128 r .. of B.  One warp
// loads (one lane), one of the leader's issues the MMAs of both CTAs (one lane), the
// kNsEpi others finish the tile from one of the two TMEM accumulators while the next
// tile is computed into the other: warp w reads lane quadrant w & 3 (32 rows) and
// the columns (1024 / kNsEpi) (w >> 2) .., 32 at a time.
struct NsBarriers {
  uint64_t full[kNsStages], empty[kNsStages], t_full[2], t_empty[2];
  uint64_t c_full[kNsEpi];
};
// What a thread carries through the tiles of a product.
struct NsCta {
  NsBarriers* b;
  uint8_t* smem;
  volatile int* abort_flag;
  uint32_t tmem;
  int rank;
  int q = 0, i = 0;  // ring uses (finishing warps: C blocks) and tiles so far
};
struct NsMaps {
  const CUtensorMap *ah, *al, *bh, *bl, *ch, *cl, *dh, *dl;
};

// The tiles first, first + step, .. < end of one product.
template <int MODE>
__device__ __forceinline__ void ns_product(NsCta& cta, const NsMaps& mp, const NsGemmParams& p,
                                           int first, int step, int end) {
  constexpr bool SYM = MODE == kNsGram || MODE == kNsPoly;
  constexpr int kStage = kNsStageBytes, kStages = kNsStages;
  constexpr int kEpi = kNsEpi;
  constexpr int kB = kStage / 2;  // B parts follow the A parts
  uint8_t* const smem = cta.smem;
  volatile int* const abort_flag = cta.abort_flag;
  const uint32_t tmem = cta.tmem;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, rank = cta.rank;
  const int nk = (p.K + 63) / 64;
  if (warp == kEpi) {
    {
      const uint32_t on = elect_lane();
      int& q = cta.q;
      bool ok = true;
      for (int u = first; ok && u < end && !__any_sync(0xffffffffu, *abort_flag); u += step) {
        const NsTile t = ns_tile<SYM>(p, u);
        const int ra = t.ti * kNsTile + rank * 128, cb = t.tj * kNsTile + rank * 128;
        for (int k = 0; k < nk; ++k, ++q) {
          const int s = q % kStages;
          if (q >= kStages && !__all_sync(0xffffffffu, mbar_wait(&cta.b->empty[s], ((q / kStages) - 1) & 1))) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kStage;
          const uint32_t bar = cluster_map(smem_u32(&cta.b->full[s]), 0);
          if (rank == 0 && on) mbar_expect_tx(&cta.b->full[s], 2 * kStage);  // both CTAs' bytes
          ns_load<true>(on, st, mp.ah, bar, 64 * k, ra, t.l);
          ns_load<true>(on, st + kNsPart, mp.al, bar, 64 * k, ra, t.l);
          if (SYM) {
            ns_load<true>(on, st + kB, mp.bh, bar, 64 * k, cb, t.l);
            ns_load<true>(on, st + kB + kNsPart, mp.bl, bar, 64 * k, cb, t.l);
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              ns_load<true>(on, st + kB + c * 8192, mp.bh, bar, cb + 64 * c, 64 * k, t.l);
              ns_load<true>(on, st + kB + kNsPart + c * 8192, mp.bl, bar, cb + 64 * c, 64 * k, t.l);
            }
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // every copy lands before shared memory goes away: the leader sees both
      // CTAs' copies, the peer stays until the cluster barrier below
      if (rank == 0)
        for (int j = q > kStages ? q - kStages : 0; j < q; ++j)
          mbar_wait(&cta.b->full[j % kStages], (j / kStages) & 1);
    }
  } else if (warp == kEpi + 1) {
    if (rank == 0) {
      const uint32_t on = elect_lane();
      const uint32_t idesc = ns_idesc(kNsTile, kNsTile, SYM ? 0 : 1);
      int &q = cta.q, &i = cta.i;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      bool ok = true;
      for (int u = first; ok && u < end && !__any_sync(0xffffffffu, *abort_flag); u += step, ++i) {
        const int b = i & 1;
        if (i >= 2 && !__all_sync(0xffffffffu, mbar_wait(&cta.b->t_empty[b], ((i >> 1) - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + b * kNsTile;
        for (int k = 0; k < nk; ++k, ++q) {
          const int s = q % kStages;
          if (!__all_sync(0xffffffffu, mbar_wait(&cta.b->full[s], (q / kStages) & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t ah = smem_u32(smem + s * kStage), bh = ah + kB;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t dah = kmaj_desc(ah, 128, ks);
            const uint64_t dbh = SYM ? kmaj_desc(bh, 128, ks) : mnmaj_desc(bh, 64, ks);
            const uint64_t dal = kmaj_desc(ah + kNsPart, 128, ks);
            const uint64_t dbl = SYM ? kmaj_desc(bh + kNsPart, 128, ks)
                                     : mnmaj_desc(bh + kNsPart, 64, ks);
            ns_umma<true>(on, acc, dal, dbh, idesc, k > 0 || ks > 0);
            ns_umma<true>(on, acc, dah, dbl, idesc, 1);
            ns_umma<true>(on, acc, dah, dbh, idesc, 1);
          }
          ns_commit<true>(on, &cta.b->empty[s]);
          last_bar = &cta.b->empty[s];
          last_par = (q / kStages) & 1;
        }
        if (!ok) break;
        ns_commit<true>(on, &cta.b->t_full[b]);
        last_bar = &cta.b->t_full[b];
        last_par = (i >> 1) & 1;
      }
      if (!ok) *abort_flag = 1;
      if (last_bar) mbar_wait(last_bar, last_par);  // all issued MMAs are done
    }
  } else {
    constexpr int kCols = 1024 / kEpi;  // of this warp
    const int quad = warp & 3, group = warp >> 2;
    uint8_t* slot = smem + kStages * kStage + warp * 2 * kNsSlot;
    const uint32_t bh = smem_u32(slot), bl = bh + kNsSlot;  // hi and lo block
    constexpr bool HAS_C = MODE != kNsGram;
    constexpr float kDown = 1.f / kNsScale;
    const float al = (MODE == kNsPoly ? p.alpha : 1.f) * kDown;
    bool stores = false;  // bulk stores issued (lane 0)
    int& cq = cta.q;        // C blocks so far
    int& i = cta.i;
    auto fetch_c = [&](int c, int r, int l) {
      if (lane == 0) {
        if (stores) bulk_wait_read_all();  // the blocks' last contents have left
        mbar_expect_tx(&cta.b->c_full[warp], 2 * kNsSlot);
        tma_load_3d(slot, mp.ch, &cta.b->c_full[warp], c, r, l);
        tma_load_3d(slot + kNsSlot, mp.cl, &cta.b->c_full[warp], c, r, l);
      }
    };
    for (int u = first; u < end; u += step, ++i) {
      const int b = i & 1;
      const NsTile t = ns_tile<SYM>(p, u);
      const int r0 = t.ti * kNsTile + rank * 128 + quad * 32;
      const int col0 = t.tj * kNsTile + group * kCols;
      const int rows = min(32, p.M - r0);  // of this warp
      const bool work = rows > 0 && col0 < p.cols;
      // C does not depend on the products: its first block is on the way while
      // they finish
      if (HAS_C && work) fetch_c(col0, r0, t.l);
      const bool got =
          __all_sync(0xffffffffu, *abort_flag == 0 && mbar_wait(&cta.b->t_full[b], (i >> 1) & 1));
      if (!got) {
        *abort_flag = 1;
        if (HAS_C && work) mbar_wait(&cta.b->c_full[warp], cq & 1);  // the copies land first
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int cc = 0; cc < kCols / 32; ++cc) {
        const int c0 = col0 + 32 * cc;
        if (!work || c0 >= p.cols) break;  // the same for the whole warp
        float v[32];
        tmem_ld32(tmem + ((quad * 32) << 16) + b * kNsTile + group * kCols + 32 * cc, v);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] *= al;
        if (HAS_C) {
          if (!__all_sync(0xffffffffu, mbar_wait(&cta.b->c_full[warp], cq & 1))) {
            *abort_flag = 1;
            break;
          }
          ++cq;
          ns_add(bh, p.beta, v);
          ns_add(bl, p.beta, v);
        } else {
          if (lane == 0 && stores) bulk_wait_read_all();
          __syncwarp();
        }
        uint32_t w[16];
        if (MODE == kNsLast) {
          if (p.tall) {
            __nv_bfloat16* o = p.out + (size_t(t.l) * p.cols + c0) * p.M + r0 + lane;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (lane < rows && c0 + e < p.cols)
                o[size_t(e) * p.M] = __float2bfloat16_rn(v[e] * kDown);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack_bf16(v[2 * e] * kDown, v[2 * e + 1] * kDown);
            ns_put(bh, w);
            __syncwarp();
            ns_store(bh, p.out + (size_t(t.l) * p.M + r0) * p.cols + c0, p.cols, rows, p.cols - c0,
                     p.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0);
          }
          fence_async_smem();  // the next C block overwrites what was read here
          __syncwarp();
        } else {
          // hi parts, then what they leave as lo parts
          ns_split_row(v, w);
          ns_put(bh, w);
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack_half2(v[2 * e], v[2 * e + 1]);
          ns_put(bl, w);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(mp.dh, slot, c0, r0, t.l);
            tma_store_3d(mp.dl, slot + kNsSlot, c0, r0, t.l);
            bulk_commit();
            stores = true;
          }
          if (SYM && t.tj < t.ti) {
            // the mirror image of a tile below the diagonal
            uint32_t m[16];
            ns_read_transposed(bh, w);
            ns_read_transposed(bl, m);
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
            ns_write_transposed(bh, w);
            ns_write_transposed(bl, m);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(mp.dh, slot, r0, c0, t.l);
              tma_store_3d(mp.dl, slot + kNsSlot, r0, c0, t.l);
              bulk_commit();
            }
          }
        }
        if (HAS_C && cc + 1 < kCols / 32 && c0 + 32 < p.cols) fetch_c(c0 + 32, r0, t.l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) cluster_arrive(cluster_map(smem_u32(&cta.b->t_empty[b]), 0));
    }
    if (lane == 0 && stores) bulk_wait_all();
  }
}

// ------------------------------------------------ matrices of at most 128 rows
// One CTA works through a matrix: all steps in one launch, with no barrier wider
// than the CTA between its products (cta_group::1, tiles of 128 x 128).  What bounds
// it is latency: a product is one or a few tiles deep, so rings and finishing warps
// are laid out for short chains.  X X^T and A A read one operand (both sides are the
// same rows), through four stages of 32 KiB; a X + B X is (a I + B) X, so that no tile
// waits for its part of X (the 22 bits of a I + B are as good as a X apart), through
// two stages of 64 KiB; each finishing warp takes one 32 x 32 block.
constexpr int kSoloEpi = 16;
constexpr int kSoloThreads = (kSoloEpi + 2) * 32;
constexpr int kSoloRing = 8 * kNsPart;
constexpr int kSoloSmem = kSoloRing + kSoloEpi * 2 * kNsSlot + 1024;
struct NsSoloBarriers {
  uint64_t full[2][4], empty[2][4];  // [ring: one operand, two operands]
  uint64_t t_full[2], t_empty[2], c_full[kSoloEpi];
};
struct NsSolo {
  NsSoloBarriers* b;
  uint8_t* smem;
  volatile int* abort_flag;
  uint32_t tmem;
  int ring[2] = {0, 0};  // uses of the rings so far
  int q = 0, i = 0;      // finishing warps: C blocks; tiles so far
};

template <int MODE>
__device__ __forceinline__ void ns_solo_product(NsSolo& cta, const NsMaps& mp, const NsGemmParams& p,
                                                int first, int step, int end) {
  constexpr bool SYM = MODE == kNsGram || MODE == kNsPoly;
  constexpr int kEpi = kSoloEpi;
  uint8_t* const smem = cta.smem;
  volatile int* const abort_flag = cta.abort_flag;
  const uint32_t tmem = cta.tmem;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nk = (p.K + 63) / 64;
  constexpr int ring = SYM ? 0 : 1, kStages = SYM ? 4 : 2;
  constexpr int kStage = (SYM ? 2 : 4) * kNsPart;
  uint64_t *const full = cta.b->full[ring], *const empty = cta.b->empty[ring];
  if (warp == kEpi) {
    {
      const uint32_t on = elect_lane();
      int& q = cta.ring[ring];
      bool ok = true;
      for (int u = first; ok && u < end && !__any_sync(0xffffffffu, *abort_flag); u += step) {
        const int l = u / p.per, col = u % p.per * 128;
        for (int k = 0; k < nk; ++k, ++q) {
          const int s = q % kStages;
          if (q >= kStages && !__all_sync(0xffffffffu, mbar_wait(&empty[s], ((q / kStages) - 1) & 1))) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kStage;
          const uint32_t bar = smem_u32(&full[s]);
          if (on) mbar_expect_tx(&full[s], kStage);
          ns_load<false>(on, st, mp.ah, bar, 64 * k, 0, l);
          ns_load<false>(on, st + kNsPart, mp.al, bar, 64 * k, 0, l);
          if (!SYM) {
            uint8_t* sb = st + 2 * kNsPart;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              ns_load<false>(on, sb + h * 8192, mp.bh, bar, col + 64 * h, 64 * k, l);
              ns_load<false>(on, sb + kNsPart + h * 8192, mp.bl, bar, col + 64 * h, 64 * k, l);
            }
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // every copy lands before shared memory is used otherwise
      for (int j = q > kStages ? q - kStages : 0; j < q; ++j)
        mbar_wait(&full[j % kStages], (j / kStages) & 1);
    }
  } else if (warp == kEpi + 1) {
    {
      const uint32_t on = elect_lane();
      const uint32_t idesc = ns_idesc(128, 128, SYM ? 0 : 1);
      int& q = cta.ring[ring];
      int& i = cta.i;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      bool ok = true;
      for (int u = first; ok && u < end && !__any_sync(0xffffffffu, *abort_flag); u += step, ++i) {
        const int b = i & 1;
        if (i >= 2 && !__all_sync(0xffffffffu, mbar_wait(&cta.b->t_empty[b], ((i >> 1) - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + b * 128;
        for (int k = 0; k < nk; ++k, ++q) {
          const int s = q % kStages;
          if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (q / kStages) & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t ah = smem_u32(smem + s * kStage), bh = SYM ? ah : ah + 2 * kNsPart;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t dah = kmaj_desc(ah, 128, ks);
            const uint64_t dbh = SYM ? dah : mnmaj_desc(bh, 64, ks);
            const uint64_t dal = kmaj_desc(ah + kNsPart, 128, ks);
            const uint64_t dbl = SYM ? dal : mnmaj_desc(bh + kNsPart, 64, ks);
            ns_umma<false>(on, acc, dal, dbh, idesc, k > 0 || ks > 0);
            ns_umma<false>(on, acc, dah, dbl, idesc, 1);
            ns_umma<false>(on, acc, dah, dbh, idesc, 1);
          }
          ns_commit<false>(on, &empty[s]);
          last_bar = &empty[s];
          last_par = (q / kStages) & 1;
        }
        if (!ok) break;
        ns_commit<false>(on, &cta.b->t_full[b]);
        last_bar = &cta.b->t_full[b];
        last_par = (i >> 1) & 1;
      }
      if (!ok) *abort_flag = 1;
      if (last_bar) mbar_wait(last_bar, last_par);  // all issued MMAs are done
    }
  } else {
    constexpr int kCols = 32;  // of this warp
    const int quad = warp & 3, group = warp >> 2;
    uint8_t* slot = smem + kSoloRing + warp * 2 * kNsSlot;
    const uint32_t bh = smem_u32(slot), bl = bh + kNsSlot;  // hi and lo block
    constexpr bool HAS_C = MODE == kNsPoly;
    constexpr float kDown = 1.f / kNsScale;
    const float al = (MODE == kNsPoly ? p.alpha : 1.f) * kDown;
    bool stores = false;  // bulk stores issued (lane 0)
    int& cq = cta.q;        // C blocks so far
    int& i = cta.i;
    auto fetch_c = [&](int c, int r, int l) {
      if (lane == 0) {
        if (stores) bulk_wait_read_all();  // the blocks' last contents have left
        mbar_expect_tx(&cta.b->c_full[warp], 2 * kNsSlot);
        tma_load_3d(slot, mp.ch, &cta.b->c_full[warp], c, r, l);
        tma_load_3d(slot + kNsSlot, mp.cl, &cta.b->c_full[warp], c, r, l);
      }
    };
    for (int u = first; u < end; u += step, ++i) {
      const int b = i & 1;
      const NsTile t{u / p.per, 0, u % p.per};
      const int r0 = quad * 32;
      const int col0 = t.tj * 128 + group * kCols;
      const int rows = min(32, p.M - r0);  // of this warp
      const bool work = rows > 0 && col0 < p.cols;
      // C does not depend on the products: its first block is on the way while
      // they finish
      if (HAS_C && work) fetch_c(col0, r0, t.l);
      const bool got =
          __all_sync(0xffffffffu, *abort_flag == 0 && mbar_wait(&cta.b->t_full[b], (i >> 1) & 1));
      if (!got) {
        *abort_flag = 1;
        if (HAS_C && work) mbar_wait(&cta.b->c_full[warp], cq & 1);  // the copies land first
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int cc = 0; cc < kCols / 32; ++cc) {
        const int c0 = col0 + 32 * cc;
        if (!work || c0 >= p.cols) break;  // the same for the whole warp
        float v[32];
        tmem_ld32(tmem + ((quad * 32) << 16) + b * 128 + group * kCols + 32 * cc, v);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] *= al;
        if (HAS_C) {
          if (!__all_sync(0xffffffffu, mbar_wait(&cta.b->c_full[warp], cq & 1))) {
            *abort_flag = 1;
            break;
          }
          ++cq;
          ns_add(bh, p.beta, v);
          ns_add(bl, p.beta, v);
          if (r0 == c0) {  // + a I
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] += e == lane ? p.diag : 0.f;
          }
        } else {
          if (lane == 0 && stores) bulk_wait_read_all();
          __syncwarp();
        }
        uint32_t w[16];
        if (MODE == kNsLast) {
          if (p.tall) {
            __nv_bfloat16* o = p.out + (size_t(t.l) * p.cols + c0) * p.M + r0 + lane;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (lane < rows && c0 + e < p.cols)
                o[size_t(e) * p.M] = __float2bfloat16_rn(v[e] * kDown);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack_bf16(v[2 * e] * kDown, v[2 * e + 1] * kDown);
            ns_put(bh, w);
            __syncwarp();
            ns_store(bh, p.out + (size_t(t.l) * p.M + r0) * p.cols + c0, p.cols, rows, p.cols - c0,
                     p.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0);
          }
          fence_async_smem();  // the next C block overwrites what was read here
          __syncwarp();
        } else {
          // hi parts, then what they leave as lo parts
          ns_split_row(v, w);
          ns_put(bh, w);
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack_half2(v[2 * e], v[2 * e + 1]);
          ns_put(bl, w);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(mp.dh, slot, c0, r0, t.l);
            tma_store_3d(mp.dl, slot + kNsSlot, c0, r0, t.l);
            bulk_commit();
            stores = true;
          }
        }
        if (HAS_C && cc + 1 < kCols / 32 && c0 + 32 < p.cols) fetch_c(c0 + 32, r0, t.l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&cta.b->t_empty[b]);
    }
    if (lane == 0 && stores) bulk_wait_all();
  }
}

__device__ __forceinline__ void ns_solo_between() {
  asm volatile("fence.proxy.async;" ::: "memory");
  __syncthreads();
  asm volatile("fence.proxy.async;" ::: "memory");
}

// Shared memory, barriers and TMEM of a CTA of a pair; all threads of both CTAs.
__device__ __forceinline__ NsCta ns_open(uint8_t* smem_raw, NsBarriers* b, uint32_t* tmem_base,
                                         int* abort_flag) {
  const int tid = threadIdx.x;
  if (tid == 0) {
    for (int i = 0; i < kNsStages; ++i) {
      mbar_init(&b->full[i], 1);
      mbar_init(&b->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b->t_full[i], 1);
      mbar_init(&b->t_empty[i], 2 * kNsEpi);
    }
    for (int i = 0; i < kNsEpi; ++i) mbar_init(&b->c_full[i], 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (tid < 32) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_base)),
                 "r"(2 * kNsTile));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are ready
  tc_fence_after();
  NsCta c;
  c.b = b;
  c.smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  c.abort_flag = abort_flag;
  c.tmem = *tmem_base;
  c.rank = int(cluster_rank());
  return c;
}
__device__ __forceinline__ void ns_close(uint32_t tmem) {
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other may signal or read it
  if (threadIdx.x < 32) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(2 * kNsTile));
  }
}

template <int MODE>
__global__ void __launch_bounds__(kNsThreads, 1)
    ns_gemm_kernel(const __grid_constant__ CUtensorMap map_ah, const __grid_constant__ CUtensorMap map_al,
                   const __grid_constant__ CUtensorMap map_bh, const __grid_constant__ CUtensorMap map_bl,
                   const __grid_constant__ NsEpiMaps em, NsGemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) NsBarriers bars;
  __shared__ uint32_t tmem_base;
  __shared__ int s_abort;
  if (threadIdx.x == 0) {
    prefetch_tmap(&map_ah);
    prefetch_tmap(&map_bh);
  }
  NsCta c = ns_open(smem_raw, &bars, &tmem_base, &s_abort);
  pdl_wait();
  pdl_trigger();
  const NsMaps m{&map_ah, &map_al, &map_bh, &map_bl, &em.ch, &em.cl, &em.dh, &em.dl};
  ns_product<MODE>(c, m, p, blockIdx.x >> 1, gridDim.x >> 1, p.nunits);
  ns_close(c.tmem);
}

struct NsAllMaps {  // [part: hi, lo], X twice
  CUtensorMap xa[2][2], xk[2][2], xe[2][2], aa[2], ae[2], ba[2], be[2];
};

__global__ void __launch_bounds__(kSoloThreads, 1)
    ns_solo_kernel(const __grid_constant__ NsAllMaps w, NsGemmParams p, int N, int steps, float a,
                   float b, float c) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) NsSoloBarriers bars;
  __shared__ uint32_t tmem_base;
  __shared__ int s_abort;
  const int tid = threadIdx.x;
  if (tid < int(sizeof(NsAllMaps) / sizeof(CUtensorMap)))
    prefetch_tmap(reinterpret_cast<const CUtensorMap*>(&w) + tid);
  if (tid == 0) {
    for (int r = 0; r < 2; ++r)
      for (int i = 0; i < 4; ++i) {
        mbar_init(&bars.full[r][i], 1);
        mbar_init(&bars.empty[r][i], 1);
      }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.t_full[i], 1);
      mbar_init(&bars.t_empty[i], kSoloEpi);
    }
    for (int i = 0; i < kSoloEpi; ++i) mbar_init(&bars.c_full[i], 1);
    s_abort = 0;
    mbar_fence_init();
  }
  if (tid < 32) {
    tmem_alloc(&tmem_base, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  NsSolo cta;
  cta.b = &bars;
  cta.smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  cta.abort_flag = &s_abort;
  cta.tmem = tmem_base;
  const int tiles = (N + 127) / 128;
  p.diag = a * kNsScale;
  for (int l = blockIdx.x; l < p.L; l += gridDim.x) {
    for (int step = 0; step < steps; ++step) {
      const int i = step & 1, last = step == steps - 1;
      p.per = 1;
      p.cols = p.M;
      p.K = N;
      const NsMaps gram{&w.xa[i][0], &w.xa[i][1], nullptr, nullptr, nullptr, nullptr, &w.ae[0], &w.ae[1]};
      ns_solo_product<kNsGram>(cta, gram, p, l, 1, l + 1);
      ns_solo_between();
      p.K = p.M;
      p.alpha = c;
      p.beta = b;
      const NsMaps poly{&w.aa[0], &w.aa[1], nullptr, nullptr, &w.ae[0], &w.ae[1], &w.be[0], &w.be[1]};
      ns_solo_product<kNsPoly>(cta, poly, p, l, 1, l + 1);
      ns_solo_between();
      p.per = tiles;
      p.cols = N;
      const NsMaps next{&w.ba[0],    &w.ba[1],    &w.xk[i][0],     &w.xk[i][1],
                        &w.xe[i][0], &w.xe[i][1], &w.xe[1 - i][0], &w.xe[1 - i][1]};
      if (last)
        ns_solo_product<kNsLast>(cta, next, p, l * tiles, 1, (l + 1) * tiles);
      else
        ns_solo_product<kNsStep>(cta, next, p, l * tiles, 1, (l + 1) * tiles);
      ns_solo_between();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid < 32) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

// Partial sums of squares: 8 entries at a time in fp32, the sums of those in 64
// bits.  Eight whose fp32 sum overflowed or may have lost squares below the
// normal range are redone in 64 bits (fp32 gradients reach 1e38).
constexpr int kNsNormParts = 64;
constexpr int kNsNormThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kNsNormThreads) ns_norm_kernel(const T* g, long long per, double* part) {
  constexpr int N = 16 / sizeof(T);
  pdl_wait();
  pdl_trigger();
  __shared__ double red[kNsNormThreads / 32];
  const T* x = g + (long long)blockIdx.y * per;
  double s = 0.0;
  const long long step = (long long)gridDim.x * kNsNormThreads;
  const long long i0 = (long long)blockIdx.x * kNsNormThreads + threadIdx.x;
  auto add = [&](const float* f, int n) {
    float q = 0.f;
    for (int i = 0; i < n; ++i) q = fmaf(f[i], f[i], q);
    if (q > 1e-30f && q < 1e30f) {
      s += double(q);
    } else {
      for (int i = 0; i < n; ++i) s += double(f[i]) * double(f[i]);
    }
  };
  const bool vector = per % N == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  if (vector) {
    const uint4* v = reinterpret_cast<const uint4*>(x);
    const long long n = per / N;
    long long i = i0;
    for (; i + 3 * step < n; i += 4 * step) {
      uint4 u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = v[i + k * step];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[N];
        LpVec<T>::unpack(u[k], f);
        add(f, N);
      }
    }
    for (; i < n; i += step) {
      float f[N];
      LpVec<T>::unpack(v[i], f);
      add(f, N);
    }
  } else {
    for (long long i = i0; i < per; i += step) {
      const float f = float(x[i]);
      add(&f, 1);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < kNsNormThreads / 32; ++w) s += red[w];
    part[blockIdx.y * kNsNormParts + blockIdx.x] = s;
  }
}

// X0 times 2^12 as an fp16 pair, transposed when G is tall: 64 x 64 tiles of G.
template <typename T>
__global__ void __launch_bounds__(256)
    ns_split_kernel(const T* g, int m, int n, const double* part, int parts, float eps, __half* xh,
                    __half* xl, long long ld, int tall) {
  pdl_wait();
  pdl_trigger();
  __shared__ float tile[64][65];
  __shared__ float s_scale[2];
  const int tid = threadIdx.x;
  if (tid < 32) {
    double s = 0.0;
    for (int i = tid; i < parts; i += 32) s += part[blockIdx.z * kNsNormParts + i];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (tid == 0) {
      // the factor as two of fp32's range: its own may be below it
      const double inv = double(kNsScale) / (sqrt(s) + double(eps));
      int e;
      const double f = frexp(inv, &e);
      s_scale[0] = float(ldexp(1.0, e / 2));
      s_scale[1] = float(ldexp(f, e - e / 2));
    }
  }
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const T* src = g + (long long)blockIdx.z * m * n;
  const bool vector = n % 8 == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  // 8 columns x 2 rows of the tile per thread
  const int tr = tid >> 3, tc = (tid & 7) * 8;
  float f[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = r0 + tr + 32 * k, c = c0 + tc;
    const T* q = src + (long long)r * n + c;
    if (vector && r < m && c < n) {
      constexpr int N = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 8 / N; ++j)
        LpVec<T>::unpack(*reinterpret_cast<const uint4*>(q + j * N), f[k] + j * N);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[k][i] = r < m && c + i < n ? float(q[i]) : 0.f;
    }
  }
  __syncthreads();
  const float a = s_scale[0], b = s_scale[1];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) f[k][i] = f[k][i] * a * b;
  if (tall) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[tr + 32 * k][tc + i] = f[k][i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) f[k][i] = tile[tc + i][tr + 32 * k];
  }
  const int M = tall ? n : m;
  const int xr = tall ? c0 : r0, xc = tall ? r0 : c0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = xr + tr + 32 * k, c = xc + tc;
    if (r >= M || c >= ld) continue;
    uint32_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      h[e] = pack_half2(f[k][2 * e], f[k][2 * e + 1]);
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
      l[e] = pack_half2(f[k][2 * e] - x.x, f[k][2 * e + 1] - x.y);
    }
    const long long o = ((long long)blockIdx.z * M + r) * ld + c;
    *reinterpret_cast<uint4*>(xh + o) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(xl + o) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// X0 itself as bf16 (no steps)
template <typename T>
__global__ void __launch_bounds__(256)
    ns_scale_kernel(const T* g, long long per, const double* part, int parts, float eps,
                    __nv_bfloat16* out) {
  pdl_wait();
  pdl_trigger();
  double s = 0.0;
  for (int i = 0; i < parts; ++i) s += part[blockIdx.y * kNsNormParts + i];
  const double inv = 1.0 / (sqrt(s) + double(eps));
  const long long at = (long long)blockIdx.y * per;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < per;
       i += (long long)gridDim.x * 256)
    out[at + i] = __float2bfloat16_rn(float(double(float(g[at + i])) * inv));
}

struct NsWork {
  double* part;
  __half *xh[2], *xl[2], *ah, *al, *bh, *bl;
  long long ldx, lda;
  int M, N;
  size_t bytes;
  NsWork(void* base, long long L, int m, int n) {
    M = m < n ? m : n;
    N = m < n ? n : m;
    ldx = (N + 7) / 8 * 8;
    lda = (M + 7) / 8 * 8;
    size_t at = 0;
    auto take = [&](size_t nbytes) {
      char* q = static_cast<char*>(base) + at;
      at += (nbytes + 255) / 256 * 256;
      return q;
    };
    part = reinterpret_cast<double*>(take(size_t(L) * kNsNormParts * 8));
    const size_t x = size_t(L) * M * ldx * 2, a = size_t(L) * M * lda * 2;
    for (int i = 0; i < 2; ++i) {
      xh[i] = reinterpret_cast<__half*>(take(x));
      xl[i] = reinterpret_cast<__half*>(take(x));
    }
    ah = reinterpret_cast<__half*>(take(a));
    al = reinterpret_cast<__half*>(take(a));
    bh = reinterpret_cast<__half*>(take(a));
    bl = reinterpret_cast<__half*>(take(a));
    bytes = at;
  }
};

// [L, rows, cols] with row stride ld; box {box_cols, box_rows, 1} of 64 columns (128-byte
// swizzle) or 32 (64-byte swizzle)
static int ns_tmap(CUtensorMap* m, const __half* base, long long L, int rows, int cols, long long ld,
                   int box_cols, int box_rows) {
  const uint64_t dims[3] = {uint64_t(cols), uint64_t(rows), uint64_t(L)};
  const uint64_t strides[2] = {uint64_t(ld) * 2, uint64_t(ld) * rows * 2};
  const uint32_t box[3] = {uint32_t(box_cols), uint32_t(box_rows), 1};
  // 16-bit elements; the type only names the fill
  return make_tmap_bf16(m, base, 3, dims, strides, box,
                        box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int MODE>
static void ns_launch(const CUtensorMap (&a)[2], const CUtensorMap (&b)[2], const CUtensorMap (&c)[2],
                      const CUtensorMap (&d)[2], NsGemmParams p, cudaStream_t s) {
  constexpr bool SYM = MODE == kNsGram || MODE == kNsPoly;
  p.tiles_m = (p.M + kNsTile - 1) / kNsTile;
  const int tiles_n = (p.cols + kNsTile - 1) / kNsTile;
  p.per = SYM ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * tiles_n;
  p.nunits = p.L * p.per;
  set_smem(ns_gemm_kernel<MODE>, kNsSmem);
  const unsigned grid = 2 * unsigned(std::min(p.nunits, 74));
  const NsEpiMaps em{c[0], c[1], d[0], d[1]};
  launch_cluster_k(ns_gemm_kernel<MODE>, grid, kNsThreads, 2, kNsSmem, s, a[0], a[1], b[0], b[1], em, p);
}

}  // namespace cyfa

extern "C" {

size_t cyfa_newton_schulz_work_bytes(int L, int m, int n) {
  return L > 0 && m > 0 && n > 0 ? NsWork(nullptr, L, m, n).bytes : 0;
}

int cyfa_newton_schulz(const void* g, int dtype, int L, int m, int n, int steps, float a, float b,
                       float c, float eps, void* out, void* work, size_t work_bytes,
                       void* stream) {
  CYFA_REQUIRE(g && out && work, kNullPointer);
  // L is also a grid dimension and a TMA coordinate
  CYFA_REQUIRE(L > 0 && L <= 65535 && m > 0 && n > 0 && m <= (1 << 16) && n <= (1 << 16) &&
                   steps >= 0 && steps <= 64,
               kBadShape);
  CYFA_REQUIRE(dtype == 0 || dtype == 1, kBadDtype);
  CYFA_REQUIRE(aligned(g, dtype == 1 ? 2 : 4) && aligned(out, 2) && aligned(work, 256), kMisaligned);
  const NsWork w(work, L, m, n);
  CYFA_REQUIRE(work_bytes >= w.bytes, kWorkspace);
  const int tiles = (w.M + 127) / 128;
  CYFA_REQUIRE((long long)L * tiles * ((w.N + 127) / 128) < (1ll << 30), kBadShape);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int tall = m > n;
  const long long per = (long long)m * n;
  const int parts = int(std::min<long long>(kNsNormParts, (per + 16383) / 16384));
  if (dtype == 1)
    CYFA_LAUNCH("ns_norm", s, (launch_k(ns_norm_kernel<__nv_bfloat16>, dim3(parts, L), kNsNormThreads, 0, s,
                                        static_cast<const __nv_bfloat16*>(g), per, w.part)));
  else
    CYFA_LAUNCH("ns_norm", s, (launch_k(ns_norm_kernel<float>, dim3(parts, L), kNsNormThreads, 0, s,
                                        static_cast<const float*>(g), per, w.part)));
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  if (steps == 0) {
    const dim3 grid(unsigned(std::min<long long>((per + 255) / 256, 1024)), L);
    if (dtype == 1)
      CYFA_LAUNCH("ns_scale", s, (launch_k(ns_scale_kernel<__nv_bfloat16>, grid, 256, 0, s,
                                           static_cast<const __nv_bfloat16*>(g), per, w.part, parts,
                                           eps, o)));
    else
      CYFA_LAUNCH("ns_scale", s, (launch_k(ns_scale_kernel<float>, grid, 256, 0, s,
                                           static_cast<const float*>(g), per, w.part, parts, eps, o)));
    return launch_status();
  }
  {
    const dim3 grid(unsigned((n + 63) / 64), unsigned((m + 63) / 64), unsigned(L));
    if (dtype == 1)
      CYFA_LAUNCH("ns_split", s, (launch_k(ns_split_kernel<__nv_bfloat16>, grid, 256, 0, s,
                                           static_cast<const __nv_bfloat16*>(g), m, n, w.part, parts,
                                           eps, w.xh[0], w.xl[0], w.ldx, tall)));
    else
      CYFA_LAUNCH("ns_split", s, (launch_k(ns_split_kernel<float>, grid, 256, 0, s,
                                           static_cast<const float*>(g), m, n, w.part, parts, eps,
                                           w.xh[0], w.xl[0], w.ldx, tall)));
  }
  // rows x 64 columns of X, A and B for the operands read along their rows, 64 x 64
  // of X for B X, where X is read down its columns
  // and 32 x 32 blocks for the finishing warps
  NsAllMaps t;
  for (int h = 0; h < 2; ++h) {
    int rc = kOk;
    for (int i = 0; i < 2 && !rc; ++i) {
      const __half* x = h ? w.xl[i] : w.xh[i];
      rc = ns_tmap(&t.xa[i][h], x, L, w.M, w.N, w.ldx, 64, 128);
      if (!rc) rc = ns_tmap(&t.xk[i][h], x, L, w.M, w.N, w.ldx, 64, 64);
      if (!rc) rc = ns_tmap(&t.xe[i][h], x, L, w.M, w.N, w.ldx, 32, 32);
    }
    const __half *a_ = h ? w.al : w.ah, *b_ = h ? w.bl : w.bh;
    if (!rc) rc = ns_tmap(&t.aa[h], a_, L, w.M, w.M, w.lda, 64, 128);
    if (!rc) rc = ns_tmap(&t.ae[h], a_, L, w.M, w.M, w.lda, 32, 32);
    if (!rc) rc = ns_tmap(&t.ba[h], b_, L, w.M, w.M, w.lda, 64, 128);
    if (!rc) rc = ns_tmap(&t.be[h], b_, L, w.M, w.M, w.lda, 32, 32);
    if (rc) return rc;
  }
  NsGemmParams q{};
  q.L = L;
  q.M = w.M;
  q.out = o;
  q.tall = tall;
  if (w.M <= 128 && (w.N <= kNsSoloWidth || L >= kNsSoloCount || w.M <= kNsSoloRows)) {
    set_smem(ns_solo_kernel, kSoloSmem);
    CYFA_LAUNCH("ns_solo", s, (launch_k(ns_solo_kernel, unsigned(std::min(L, 148)), kSoloThreads,
                                        kSoloSmem, s, t, q, w.N, steps, a, b, c)));
    return launch_status();
  }
  for (int step = 0; step < steps; ++step) {
    const int i = step & 1, last = step == steps - 1;
    NsGemmParams p = q;
    p.cols = w.M;
    p.K = w.N;
    CYFA_LAUNCH("ns_gram", s, (ns_launch<kNsGram>(t.xa[i], t.xa[i], t.ae, t.ae, p, s)));
    p.K = w.M;
    p.alpha = c;
    p.beta = b;
    CYFA_LAUNCH("ns_poly", s, (ns_launch<kNsPoly>(t.aa, t.aa, t.ae, t.be, p, s)));
    p.cols = w.N;
    p.beta = a;
    if (last)
      CYFA_LAUNCH("ns_last", s, (ns_launch<kNsLast>(t.ba, t.xk[i], t.xe[i], t.xe[i], p, s)));
    else
      CYFA_LAUNCH("ns_step", s, (ns_launch<kNsStep>(t.ba, t.xk[i], t.xe[i], t.xe[1 - i], p, s)));
  }
  return launch_status();
}

}  // extern "C"
