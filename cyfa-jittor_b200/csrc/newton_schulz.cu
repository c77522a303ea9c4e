// Newton-Schulz orthogonalisation of a batch of matrices G [m, n] (the update of
// the Muon optimiser): with X0 = G / (|G|_F + eps), taken as [M, N], M <= N
// (transposed when G is tall),
//   A = X X^T,   B = b A + c A A,   X <- a X + B X        (each step)
// which pushes every singular value towards 1.
//
// The products run on tcgen05 with fp32 accumulators in TMEM.  Small singular
// values grow by a = 3.4 a step, and so do rounding errors beside them, so the
// operands are kept as fp16 pairs hi + lo (22 significant bits) and a product is
// the three MMAs hi hi + hi lo + lo hi.  X, A and B are stored times 2^12, which
// keeps the lo parts of small entries above fp16's underflow and leaves room up
// to |entry| < 16.  A and B are symmetric: only the tiles on and below the
// diagonal are computed, the others are written as their mirror images.
#include <cuda_fp16.h>

#include "cyfa_common.cuh"

namespace cyfa {

constexpr float kNsScale = 4096.f;  // 2^12
constexpr int kNsEpiWarps = 8;
constexpr int kNsThreads = (kNsEpiWarps + 2) * 32;

enum NsMode : int {
  kNsGram = 0,    // D = acc
  kNsPoly = 1,    // D = alpha acc + beta C
  kNsStep = 2,    // D = acc + beta C, row-major
  kNsLast = 3,    // the step's result as bf16, in G's orientation
};

struct NsGemmParams {
  int L, M, cols, K;        // D [L, M, cols] = contraction over K
  int tiles_m, tiles_n;
  float alpha, beta;
  const __half *ch, *cl;    // C pair, layout of D
  __half *dh, *dl;          // D pair [L, M, ld]
  long long ld;             // row stride of C and D (a multiple of 8)
  __nv_bfloat16* out;       // kNsLast
  int tall;                 // out is [L, cols, M]
};

template <int BN>
constexpr int ns_stage_bytes() {
  return 2 * 128 * 128 + 2 * BN * 128;  // Ah, Al [128 x 64], Bh, Bl [BN x 64]
}
template <int BN>
constexpr int ns_stages() {
  return BN == 256 ? 2 : 3;
}
template <int BN>
constexpr int ns_smem() {
  return ns_stages<BN>() * ns_stage_bytes<BN>() + 1024;
}

// fp16 x fp16 -> fp32
__host__ __device__ constexpr uint32_t ns_idesc(int M, int N, int b_mn) {
  return (1u << 4) | (uint32_t(b_mn) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

// Unit u -> (matrix, row tile, column tile).  Symmetric products skip the tiles
// above the diagonal: row tile i has the column tiles j with j BN/128 <= i.
struct NsTile {
  int l, ti, tj;
};
template <int BN, bool SYM>
__device__ __forceinline__ NsTile ns_tile(const NsGemmParams& p, int u, int per) {
  NsTile t;
  t.l = u / per;
  int r = u - t.l * per;
  if (SYM) {
    constexpr int nb = BN / 128;
    t.ti = 0;
    while (true) {
      const int w = t.ti / nb + 1;
      if (r < w) break;
      r -= w;
      ++t.ti;
    }
    t.tj = r;
  } else {
    t.ti = r % p.tiles_m;
    t.tj = r / p.tiles_m;
  }
  return t;
}

__device__ __forceinline__ uint32_t pack_half2(__half a, __half b) {
  return uint32_t(__half_as_ushort(a)) | (uint32_t(__half_as_ushort(b)) << 16);
}

// Persistent; warp 8 loads (one lane), warp 9 issues the MMAs (one lane), warps
// 0-7 finish tiles from the two TMEM accumulators: warp w reads lane quadrant
// w & 3 (32 rows) and column half w >> 2.
template <int BN, int MODE>
__global__ void __launch_bounds__(kNsThreads, 1)
    ns_gemm_kernel(const __grid_constant__ CUtensorMap map_ah, const __grid_constant__ CUtensorMap map_al,
                   const __grid_constant__ CUtensorMap map_bh, const __grid_constant__ CUtensorMap map_bl,
                   NsGemmParams p, int nunits, int per) {
  constexpr bool SYM = MODE == kNsGram || MODE == kNsPoly;
  constexpr int kStage = ns_stage_bytes<BN>(), kStages = ns_stages<BN>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], t_full[2], t_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int s_abort;
  volatile int* abort_flag = &s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], kNsEpiWarps);
    }
    s_abort = 0;
    mbar_fence_init();
    prefetch_tmap(&map_ah);
    prefetch_tmap(&map_al);
    prefetch_tmap(&map_bh);
    prefetch_tmap(&map_bl);
  }
  if (warp == 0) {
    tmem_alloc(&tmem_base, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = tmem_base;
  const int nk = (p.K + 63) / 64;

  if (warp == kNsEpiWarps) {
    if (lane == 0) {
      int q = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < nunits && !*abort_flag; u += gridDim.x) {
        const NsTile t = ns_tile<BN, SYM>(p, u, per);
        for (int k = 0; k < nk; ++k, ++q) {
          const int s = q % kStages;
          if (q >= kStages && !mbar_wait(&empty[s], ((q / kStages) - 1) & 1)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kStage;
          mbar_expect_tx(&full[s], kStage);
          tma_load_3d(st, &map_ah, &full[s], 64 * k, t.ti * 128, t.l);
          tma_load_3d(st + 16384, &map_al, &full[s], 64 * k, t.ti * 128, t.l);
          uint8_t* sb = st + 32768;
          if (SYM) {
            tma_load_3d(sb, &map_bh, &full[s], 64 * k, t.tj * BN, t.l);
            tma_load_3d(sb + BN * 128, &map_bl, &full[s], 64 * k, t.tj * BN, t.l);
          } else {
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) {
              tma_load_3d(sb + c * 8192, &map_bh, &full[s], t.tj * BN + 64 * c, 64 * k, t.l);
              tma_load_3d(sb + BN * 128 + c * 8192, &map_bl, &full[s], t.tj * BN + 64 * c, 64 * k,
                          t.l);
            }
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // every issued copy lands before shared memory goes away
      for (int j = q > kStages ? q - kStages : 0; j < q; ++j)
        mbar_wait(&full[j % kStages], (j / kStages) & 1);
    }
  } else if (warp == kNsEpiWarps + 1) {
    if (lane == 0) {
      const uint32_t idesc = ns_idesc(128, BN, SYM ? 0 : 1);
      int q = 0, i = 0;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < nunits && !*abort_flag; u += gridDim.x, ++i) {
        const int b = i & 1;
        if (i >= 2 && !mbar_wait(&t_empty[b], ((i >> 1) - 1) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + b * BN;
        for (int k = 0; k < nk; ++k, ++q) {
          const int s = q % kStages;
          if (!mbar_wait(&full[s], (q / kStages) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t ah = smem_u32(smem + s * kStage), al = ah + 16384, bh = ah + 32768,
                         bl = bh + BN * 128;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t dah = kmaj_desc(ah, 128, ks), dal = kmaj_desc(al, 128, ks);
            const uint64_t dbh = SYM ? kmaj_desc(bh, BN, ks) : mnmaj_desc(bh, 64, ks);
            const uint64_t dbl = SYM ? kmaj_desc(bl, BN, ks) : mnmaj_desc(bl, 64, ks);
            umma_bf16(acc, dal, dbh, idesc, k > 0 || ks > 0);
            umma_bf16(acc, dah, dbl, idesc, 1);
            umma_bf16(acc, dah, dbh, idesc, 1);
          }
          umma_commit(&empty[s]);
          last_bar = &empty[s];
          last_par = (q / kStages) & 1;
        }
        if (!ok) break;
        umma_commit(&t_full[b]);
        last_bar = &t_full[b];
        last_par = (i >> 1) & 1;
      }
      if (!ok) *abort_flag = 1;
      if (last_bar) mbar_wait(last_bar, last_par);  // all issued MMAs are done
    }
  } else {
    const int quad = warp & 3, half = warp >> 2;
    int i = 0;
    for (int u = blockIdx.x; u < nunits; u += gridDim.x, ++i) {
      const int b = i & 1;
      const bool got =
          __all_sync(0xffffffffu, *abort_flag == 0 && mbar_wait(&t_full[b], (i >> 1) & 1));
      if (!got) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const NsTile t = ns_tile<BN, SYM>(p, u, per);
      const int r = t.ti * 128 + quad * 32 + lane;
      const bool row_in = r < p.M;
      const size_t mat = size_t(t.l) * p.M * p.ld;
      constexpr int nb = BN / 128;
#pragma unroll 1
      for (int cc = 0; cc < BN / 64; ++cc) {
        const int cl0 = half * (BN / 2) + 32 * cc;  // column in the tile
        const int c0 = t.tj * BN + cl0;
        float v[32];
        tmem_ld32(tmem + ((quad * 32) << 16) + b * BN + cl0, v);
        if (c0 >= p.cols) continue;  // the same for the whole warp
        const size_t row_at = mat + size_t(row_in ? r : 0) * p.ld + c0;
        if (MODE == kNsGram) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] *= 1.f / kNsScale;
        } else {
          const float al = MODE == kNsPoly ? p.alpha / kNsScale : 1.f / kNsScale;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (row_in && c0 + 8 * g < p.ld) {
              const uint4 uh = *reinterpret_cast<const uint4*>(p.ch + row_at + 8 * g);
              const uint4 ul = *reinterpret_cast<const uint4*>(p.cl + row_at + 8 * g);
              const __half2* hh = reinterpret_cast<const __half2*>(&uh);
              const __half2* hl = reinterpret_cast<const __half2*>(&ul);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x = __half22float2(hh[e]), y = __half22float2(hl[e]);
                v[8 * g + 2 * e] = fmaf(p.beta, x.x + y.x, v[8 * g + 2 * e] * al);
                v[8 * g + 2 * e + 1] = fmaf(p.beta, x.y + y.y, v[8 * g + 2 * e + 1] * al);
              }
            }
          }
        }
        if (MODE == kNsLast) {
          if (p.tall) {
            __nv_bfloat16* o = p.out + size_t(t.l) * p.cols * p.M + size_t(c0) * p.M + r;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (row_in && c0 + e < p.cols)
                o[size_t(e) * p.M] = __float2bfloat16_rn(v[e] * (1.f / kNsScale));
          } else if (row_in) {
            __nv_bfloat16* o = p.out + (size_t(t.l) * p.M + r) * p.cols + c0;
            if (p.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0) {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                if (c0 + 8 * g < p.cols) {
                  uint32_t w[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    w[e] = pack_bf16(v[8 * g + 2 * e] * (1.f / kNsScale),
                                     v[8 * g + 2 * e + 1] * (1.f / kNsScale));
                  *reinterpret_cast<uint4*>(o + 8 * g) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (c0 + e < p.cols) o[e] = __float2bfloat16_rn(v[e] * (1.f / kNsScale));
            }
          }
        } else {
          __half hi[32], lo[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            hi[e] = __float2half_rn(v[e]);
            lo[e] = __float2half_rn(v[e] - __half2float(hi[e]));
          }
          if (row_in) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
              if (c0 + 8 * g < p.ld) {
                uint32_t wh[4], wl[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  wh[e] = pack_half2(hi[8 * g + 2 * e], hi[8 * g + 2 * e + 1]);
                  wl[e] = pack_half2(lo[8 * g + 2 * e], lo[8 * g + 2 * e + 1]);
                }
                *reinterpret_cast<uint4*>(p.dh + row_at + 8 * g) = make_uint4(wh[0], wh[1], wh[2], wh[3]);
                *reinterpret_cast<uint4*>(p.dl + row_at + 8 * g) = make_uint4(wl[0], wl[1], wl[2], wl[3]);
              }
          }
          // the mirror image, where no tile of its own computes it
          if (SYM && c0 / 128 < t.ti / nb * nb && row_in) {
            const size_t at = mat + size_t(c0) * p.ld + r;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              p.dh[at + size_t(e) * p.ld] = hi[e];
              p.dl[at + size_t(e) * p.ld] = lo[e];
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&t_empty[b]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * BN);
  }
}

// Partial sums of squares, in 64 bits: fp32 gradients may be as large as 1e38.
constexpr int kNsNormParts = 64;
template <typename T>
__global__ void __launch_bounds__(256) ns_norm_kernel(const T* g, long long per, double* part) {
  pdl_wait();
  pdl_trigger();
  __shared__ double red[8];
  const T* x = g + (long long)blockIdx.y * per;
  double s = 0.0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < per;
       i += (long long)gridDim.x * 256) {
    const double v = double(float(x[i]));
    s += v * v;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < 8; ++w) s += red[w];
    part[blockIdx.y * kNsNormParts + blockIdx.x] = s;
  }
}

// X0 times 2^12 as an fp16 pair, transposed when G is tall: 32 x 32 tiles of G.
template <typename T>
__global__ void __launch_bounds__(256)
    ns_split_kernel(const T* g, int m, int n, const double* part, int parts, float eps, __half* xh,
                    __half* xl, long long ld, int tall) {
  pdl_wait();
  pdl_trigger();
  __shared__ float tile[32][33];
  __shared__ double s_inv;
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < parts; ++i) s += part[blockIdx.z * kNsNormParts + i];
    s_inv = double(kNsScale) / (sqrt(s) + double(eps));
  }
  __syncthreads();
  const double inv = s_inv;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
  const T* src = g + (long long)blockIdx.z * m * n;
  const int M = tall ? n : m, N = tall ? m : n;
  __half* oh = xh + (long long)blockIdx.z * M * ld;
  __half* ol = xl + (long long)blockIdx.z * M * ld;
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + ty + 8 * k, c = c0 + tx;
    const float v = r < m && c < n ? float(double(float(src[(long long)r * n + c])) * inv) : 0.f;
    if (tall) {
      tile[ty + 8 * k][tx] = v;
    } else if (r < M && c < N) {
      const __half hi = __float2half_rn(v);
      oh[(long long)r * ld + c] = hi;
      ol[(long long)r * ld + c] = __float2half_rn(v - __half2float(hi));
    }
  }
  if (!tall) return;
  __syncthreads();
  for (int k = 0; k < 4; ++k) {
    const int r = c0 + ty + 8 * k, c = r0 + tx;  // of X
    if (r < M && c < N) {
      const float v = tile[tx][ty + 8 * k];
      const __half hi = __float2half_rn(v);
      oh[(long long)r * ld + c] = hi;
      ol[(long long)r * ld + c] = __float2half_rn(v - __half2float(hi));
    }
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

// [L, rows, cols] with row stride ld; box {64, box_rows, 1}
static int ns_tmap(CUtensorMap* m, const __half* base, long long L, int rows, int cols, long long ld,
                   int box_rows) {
  const uint64_t dims[3] = {uint64_t(cols), uint64_t(rows), uint64_t(L)};
  const uint64_t strides[2] = {uint64_t(ld) * 2, uint64_t(ld) * rows * 2};
  const uint32_t box[3] = {64, uint32_t(box_rows), 1};
  return make_tmap_bf16(m, base, 3, dims, strides, box);  // 16-bit elements; the type only names the fill
}

template <int BN, int MODE>
static void ns_launch(const CUtensorMap& ah, const CUtensorMap& al, const CUtensorMap& bh,
                      const CUtensorMap& bl, NsGemmParams p, cudaStream_t s) {
  constexpr bool SYM = MODE == kNsGram || MODE == kNsPoly;
  constexpr int nb = BN / 128;
  p.tiles_m = (p.M + 127) / 128;
  p.tiles_n = (p.cols + BN - 1) / BN;
  int per = p.tiles_m * p.tiles_n;
  if (SYM) {
    per = 0;
    for (int i = 0; i < p.tiles_m; ++i) per += i / nb + 1;
  }
  const int nunits = p.L * per;
  set_smem(ns_gemm_kernel<BN, MODE>, ns_smem<BN>());
  const unsigned grid = unsigned(std::min(nunits, 148));
  launch_k(ns_gemm_kernel<BN, MODE>, grid, kNsThreads, ns_smem<BN>(), s, ah, al, bh, bl, p, nunits,
           per);
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
  const int parts = int(std::min<long long>(kNsNormParts, (per + 4095) / 4096));
  if (dtype == 1)
    CYFA_LAUNCH("ns_norm", s, (launch_k(ns_norm_kernel<__nv_bfloat16>, dim3(parts, L), 256, 0, s,
                                        static_cast<const __nv_bfloat16*>(g), per, w.part)));
  else
    CYFA_LAUNCH("ns_norm", s, (launch_k(ns_norm_kernel<float>, dim3(parts, L), 256, 0, s,
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
    const dim3 grid(unsigned((n + 31) / 32), unsigned((m + 31) / 32), unsigned(L));
    if (dtype == 1)
      CYFA_LAUNCH("ns_split", s, (launch_k(ns_split_kernel<__nv_bfloat16>, grid, 256, 0, s,
                                           static_cast<const __nv_bfloat16*>(g), m, n, w.part, parts,
                                           eps, w.xh[0], w.xl[0], w.ldx, tall)));
    else
      CYFA_LAUNCH("ns_split", s, (launch_k(ns_split_kernel<float>, grid, 256, 0, s,
                                           static_cast<const float*>(g), m, n, w.part, parts, eps,
                                           w.xh[0], w.xl[0], w.ldx, tall)));
  }
  constexpr int BN = 256;
  CUtensorMap xa[2][2], xb[2][2], xk[2][2], aa[2], ab[2], ba[2];
  for (int i = 0; i < 2; ++i)
    for (int h = 0; h < 2; ++h) {
      const __half* x = h ? w.xl[i] : w.xh[i];
      int rc = ns_tmap(&xa[i][h], x, L, w.M, w.N, w.ldx, 128);
      if (!rc) rc = ns_tmap(&xb[i][h], x, L, w.M, w.N, w.ldx, BN);
      if (!rc) rc = ns_tmap(&xk[i][h], x, L, w.M, w.N, w.ldx, 64);
      if (rc) return rc;
    }
  for (int h = 0; h < 2; ++h) {
    int rc = ns_tmap(&aa[h], h ? w.al : w.ah, L, w.M, w.M, w.lda, 128);
    if (!rc) rc = ns_tmap(&ab[h], h ? w.al : w.ah, L, w.M, w.M, w.lda, BN);
    if (!rc) rc = ns_tmap(&ba[h], h ? w.bl : w.bh, L, w.M, w.M, w.lda, 128);
    if (rc) return rc;
  }
  for (int step = 0; step < steps; ++step) {
    const int i = step & 1, last = step == steps - 1;
    NsGemmParams p{};
    p.L = L;
    p.M = w.M;
    p.out = o;
    p.tall = tall;
    p.cols = w.M;
    p.ld = w.lda;
    p.K = w.N;
    p.dh = w.ah;
    p.dl = w.al;
    CYFA_LAUNCH("ns_gram", s, (ns_launch<BN, kNsGram>(xa[i][0], xa[i][1], xb[i][0], xb[i][1], p, s)));
    p.K = w.M;
    p.alpha = c;
    p.beta = b;
    p.ch = w.ah;
    p.cl = w.al;
    p.dh = w.bh;
    p.dl = w.bl;
    CYFA_LAUNCH("ns_poly", s, (ns_launch<BN, kNsPoly>(aa[0], aa[1], ab[0], ab[1], p, s)));
    p.cols = w.N;
    p.ld = w.ldx;
    p.beta = a;
    p.ch = w.xh[i];
    p.cl = w.xl[i];
    p.dh = w.xh[1 - i];
    p.dl = w.xl[1 - i];
    if (last)
      CYFA_LAUNCH("ns_last", s, (ns_launch<BN, kNsLast>(ba[0], ba[1], xk[i][0], xk[i][1], p, s)));
    else
      CYFA_LAUNCH("ns_step", s, (ns_launch<BN, kNsStep>(ba[0], ba[1], xk[i][0], xk[i][1], p, s)));
  }
  return launch_status();
}

}  // extern "C"
