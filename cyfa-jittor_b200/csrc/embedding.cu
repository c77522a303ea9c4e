// Embedding lookup with a scale, and the gradient of the whole table.
//   out[n] = scale W[id_n]
//   dW[v]  = scale sum over {n : id_n = v} of dout[n], fp32
// The sum runs over the tokens sorted by id (a stable radix sort, so equal ids
// keep their order), in a fixed tree: up to 32 neighbours in ascending n, the partial
// sums of a longer run in eight stretches side by side, the stretches in order.  No float
// atomics, the same bits on every run.  A token
// outside the vocabulary sets the device error word, reads as a zero row and
// has no gradient; the padding row's gradient is zero.
// Bound by memory: the lookup of 16384 rows of 1024 bf16 takes 8 us (67 MB), 30011 of
// 1001 f32 28 us (240 MB, the last of it left in L2).
// The gradient of the same lookups: the sort beside the clearing of the table (15 and
// 66 us; the table's 66 and 400 MB), the sums (9 and 33; 59 and 200 MB) and the join of
// the runs that cross pieces (8 and 22, latency).
#include <algorithm>
#include <type_traits>

#include "cyfa_common.cuh"

namespace cyfa {

constexpr int kEmbThreads = 256;

// VEC elements per access; the widest that divides D and fits the pointers.
template <typename T, int VEC>
struct EmbVec {
  typedef typename std::conditional<
      sizeof(T) * VEC == 16, uint4,
      typename std::conditional<
          sizeof(T) * VEC == 8, uint2,
          typename std::conditional<sizeof(T) * VEC == 4, uint32_t, uint16_t>::type>::type>::type U;
  static __device__ __forceinline__ void load(const T* p, float* f) {
    const U u = *reinterpret_cast<const U*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = float(e[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float* f) {
    U u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = T(f[i]);
    *reinterpret_cast<U*>(p) = u;
  }
};

// CTA: kEmbItems accesses of VEC elements in a row-major walk over the output; a
// thread's accesses are all in flight together.
template <int VEC>
constexpr int emb_unroll() {
  return VEC >= 4 ? 4 : 8;
}
template <typename T, int VEC>
__global__ void __launch_bounds__(kEmbThreads)
    embed_fwd_kernel(const long long* tokens, const T* w, T* out, long long N, long long V, int D,
                     float scale) {
  constexpr int U = emb_unroll<VEC>();
  pdl_wait();
  pdl_trigger();
  const unsigned per_row = unsigned(D / VEC);
  const long long first = (long long)blockIdx.x * (U * kEmbThreads), n0 = first / per_row;
  const unsigned rem = unsigned(first - n0 * per_row);
  float f[U][VEC];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const unsigned i = rem + k * kEmbThreads + threadIdx.x, r = i / per_row;
    const long long n = n0 + r;
    const unsigned c = (i - r * per_row) * VEC;
    if (n < N) {
      const long long id = __ldg(tokens + n);
      if (id >= 0 && id < V) {
        EmbVec<T, VEC>::load(w + id * D + c, f[k]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[k][e] *= scale;
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[k][e] = 0.f;
        if (c == 0) set_error(kErrBadIndex);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const long long i = first + k * kEmbThreads + threadIdx.x;
    if (i < N * per_row) EmbVec<T, VEC>::store(out + i * VEC, f[k]);
  }
}

// The same for long rows: a warp takes 32 emb_unroll accesses of one row, so that the
// row, its token and the addresses cost nothing per access.
template <typename T, int VEC>
__global__ void __launch_bounds__(kEmbThreads)
    embed_fwd_rows_kernel(const long long* tokens, const T* w, T* out, long long N, long long V, int D,
                          float scale, int parts) {
  constexpr int U = emb_unroll<VEC>();
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * (kEmbThreads / 32) + (threadIdx.x >> 5);
  const long long n = parts == 1 ? unit : unit / parts;
  if (n >= N) return;
  const int c0 = (int(unit - n * parts) * (32 * U) + lane) * VEC;
  const long long id = __ldg(tokens + n);
  const bool ok = id >= 0 && id < V;
  const T* src = w + (ok ? id * D : 0);
  T* dst = out + n * D;
  float f[U][VEC];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int c = c0 + k * 32 * VEC;
    if (ok && c < D) {
      EmbVec<T, VEC>::load(src + c, f[k]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[k][e] = 0.f;
    }
  }
  if (!ok && c0 == 0) set_error(kErrBadIndex);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int c = c0 + k * 32 * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[k][e] *= scale;
    if (c < D) EmbVec<T, VEC>::store(dst + c, f[k]);
  }
}

// ------------------------------------------------------------------- the sort
// Stable radix sort of (id, position), 8 bits a pass.  A CTA takes kSortTile
// consecutive entries, each of its warps a run of them; ranks inside a run come
// from match masks, across runs and tiles from counts per digit.
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 16;  // entries of a lane
constexpr int kSortTile = kSortThreads * kSortRounds;

__device__ __forceinline__ uint32_t sort_key(const long long* tokens, long long V, long long pad,
                                             long long n) {
  const long long id = tokens[n];
  return id >= 0 && id < V && id != pad ? uint32_t(id) : uint32_t(V);  // dropped ids come last
}

// first pass: keys from the tokens, positions from the index
struct SortPass {
  const long long* tokens;  // first pass, else null
  const uint32_t* key_in;
  const uint32_t* pos_in;
  uint32_t* key_out;
  uint32_t* pos_out;
  uint32_t* count;  // [256][tiles]
  long long N, V, pad;
  int shift, tiles;
};

__device__ __forceinline__ uint32_t pass_key(const SortPass& p, long long n) {
  return p.tokens ? sort_key(p.tokens, p.V, p.pad, n) : p.key_in[n];
}

__global__ void __launch_bounds__(kSortThreads) embed_sort_count_kernel(SortPass p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t hist[256];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const long long n0 = (long long)blockIdx.x * kSortTile;
  for (int i = threadIdx.x; i < kSortTile; i += kSortThreads)
    if (n0 + i < p.N) atomicAdd(&hist[(pass_key(p, n0 + i) >> p.shift) & 255], 1u);
  __syncthreads();
  p.count[(size_t)threadIdx.x * p.tiles + blockIdx.x] = hist[threadIdx.x];
}

// exclusive scan of count[256 * tiles], one CTA
__global__ void __launch_bounds__(1024) embed_sort_scan_kernel(uint32_t* count, int n) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t part[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (n + 1023) / 1024, b = min(n, tid * per), e = min(n, b + per);
  uint32_t sum = 0;
  for (int i = b; i < e; ++i) sum += count[i];
  uint32_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  uint32_t before = inc - sum;
  for (int w = 0; w < warp; ++w) before += part[w];
  for (int i = b; i < e; ++i) {
    const uint32_t v = count[i];
    count[i] = before;
    before += v;
  }
}

__global__ void __launch_bounds__(kSortThreads) embed_sort_move_kernel(SortPass p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t next[kSortWarps][256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kSortWarps * 256; i += kSortThreads) (&next[0][0])[i] = 0;
  __syncthreads();
  const long long n0 = (long long)blockIdx.x * kSortTile + warp * (32 * kSortRounds);
  uint32_t key[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const long long n = n0 + r * 32 + lane;
    const bool in = n < p.N;
    key[r] = in ? pass_key(p, n) : 0u;
    const unsigned same =
        __match_any_sync(0xffffffffu, in ? (key[r] >> p.shift) & 255u : 256u);
    if (in && lane == __ffs(same) - 1) next[warp][(key[r] >> p.shift) & 255] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  {
    uint32_t run = p.count[(size_t)tid * p.tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = next[w][tid];
      next[w][tid] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const long long n = n0 + r * 32 + lane;
    const bool in = n < p.N;
    const uint32_t d = (key[r] >> p.shift) & 255u;
    const unsigned same = __match_any_sync(0xffffffffu, in ? d : 256u);
    if (in) {
      const uint32_t at = next[warp][d] + __popc(same & ((1u << lane) - 1));
      p.key_out[at] = key[r];
      p.pos_out[at] = p.pos_in ? p.pos_in[n] : uint32_t(n);
    }
    __syncwarp();
    if (in && lane == __ffs(same) - 1) next[warp][d] += __popc(same);
    __syncwarp();
  }
}

// The whole sort in one cluster of 8 CTAs, for up to kCsMax tokens: the entries live
// in the CTAs' shared memory, a thread holds its own in registers while a pass
// scatters them to their places, in whichever CTA.  A pass takes three cluster
// barriers instead of three launches.  The grid's other clusters clear the
// table's gradient meanwhile.  (The whole gradient of 64 f32 columns and 32000 rows
// against the sort by launches above: 256 tokens 17 us against 38, 16384 28 against 66,
// 65536 60 against 79, 131072 101 against 98; 300000 rows, 131072 tokens 122 against 134.)
constexpr int kCsCtas = 8;
constexpr int kCsThreads = 1024;
constexpr int kCsWarps = kCsThreads / 32;
constexpr int kCsDigits = 512;
constexpr int kCsClear = 2048;   // vectors of one clearing copy
constexpr int kCsMaxPer = 16;  // entries of a thread
constexpr long long kCsMax = (long long)kCsCtas * kCsThreads * kCsMaxPer;

struct ClusterSortParams {
  const long long* tokens;
  uint32_t *key_out, *pos_out;
  long long N, V, pad;
  int bits, passes;       // digit width, passes
  uint4* clear;           // table gradient from its first 16-byte boundary
  long long clear_vecs;
  uint8_t *edge0, *edge1;  // bytes before and after
  int edge0_bytes, edge1_bytes;
};

__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}
template <int PER>
constexpr int cs_smem() {
  return kCsThreads * PER * 8 + kCsWarps * kCsDigits * 2 + kCsDigits * 8 + 64 * 4;
}

template <int PER>
__global__ void __launch_bounds__(kCsThreads) embed_cluster_sort_kernel(ClusterSortParams p) {
  constexpr int kChunk = kCsThreads * PER;
  extern __shared__ __align__(16) uint8_t cs_smem_raw[];
  uint2* entry = reinterpret_cast<uint2*>(cs_smem_raw);                       // [kChunk] key, position
  uint16_t* run = reinterpret_cast<uint16_t*>(entry + kChunk);                // [warps][digits]
  uint32_t* count = reinterpret_cast<uint32_t*>(run + kCsWarps * kCsDigits);  // [digits] of this CTA
  uint32_t* base = count + kCsDigits;                                         // [digits]
  uint32_t* part = base + kCsDigits;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (blockIdx.x >= kCsCtas) {
    const long long i0 = (long long)(blockIdx.x - kCsCtas) * kCsThreads + tid;
    const long long step = (long long)(gridDim.x - kCsCtas) * kCsThreads;
    // 32 KiB of zeros in shared memory, stored over and over by bulk copies
    uint4* zeros = reinterpret_cast<uint4*>(cs_smem_raw);
    for (int i = tid; i < kCsClear; i += kCsThreads) zeros[i] = make_uint4(0, 0, 0, 0);
    fence_async_smem();
    __syncthreads();
    if (tid == 0) {
      for (long long v = (i0 / kCsThreads) * kCsClear; v < p.clear_vecs;
           v += (step / kCsThreads) * kCsClear)
        bulk_store(p.clear + v, zeros, uint32_t(min((long long)kCsClear, p.clear_vecs - v)) * 16);
      bulk_commit();
      bulk_wait_all();
    }
    if (i0 < p.edge0_bytes) p.edge0[i0] = 0;
    if (i0 < p.edge1_bytes) p.edge1[i0] = 0;
    return;
  }
  const uint32_t rank = cluster_rank();
  const uint32_t mask = (1u << p.bits) - 1, ndig = 1u << p.bits;
  // warp w of CTA r holds the entries (r 32 + w) 32 PER .., in rounds of 32
  const long long n0 = (long long)rank * kChunk + warp * (32 * PER) + lane;
  uint2 e[PER];
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const long long n = n0 + r * 32;
    // past the end: after every key
    e[r] = n < p.N ? make_uint2(sort_key(p.tokens, p.V, p.pad, n), uint32_t(n))
                   : make_uint2(0xffffffffu, 0xffffffffu);
  }
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    for (uint32_t d = lane; d < ndig; d += 32) run[warp * kCsDigits + d] = 0;
    __syncwarp();
    uint16_t before[PER];  // entries of the digit earlier in the warp's run
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      const uint32_t d = (e[r].x >> shift) & mask;
      const unsigned same = __match_any_sync(0xffffffffu, d);
      const uint16_t c = run[warp * kCsDigits + d];
      before[r] = uint16_t(c + __popc(same & ((1u << lane) - 1)));
      __syncwarp();
      if (lane == __ffs(same) - 1) run[warp * kCsDigits + d] = uint16_t(c + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    // runs' offsets inside the CTA, and the CTA's count, per digit
    if (tid < int(ndig)) {
      uint32_t sum = 0;
#pragma unroll 8
      for (int w = 0; w < kCsWarps; ++w) {
        const uint32_t c = run[w * kCsDigits + tid];
        run[w * kCsDigits + tid] = uint16_t(sum);
        sum += c;
      }
      count[tid] = sum;
    }
    cluster_sync_all();  // the counts are there, and every entry is in registers
    {
      uint32_t total = 0, mine = 0;
      if (tid < int(ndig)) {
#pragma unroll
        for (uint32_t c = 0; c < kCsCtas; ++c) {
          const uint32_t v = cluster_ld_u32(cluster_map(smem_u32(count + tid), c));
          if (c < rank) mine += v;
          total += v;
        }
      }
      uint32_t inc = total;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) part[warp] = inc;
      __syncthreads();
      if (warp == 0) {
        const uint32_t v = part[lane];
        uint32_t s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += t;
        }
        part[lane] = s - v;
      }
      __syncthreads();
      if (tid < int(ndig)) base[tid] = part[warp] + inc - total + mine;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      const uint32_t d = (e[r].x >> shift) & mask;
      const uint32_t at = base[d] + run[warp * kCsDigits + d] + before[r];
      cluster_st_u2(cluster_map(smem_u32(entry + at % kChunk), at / kChunk), e[r]);
    }
    cluster_sync_all();  // every entry is in its place
#pragma unroll
    for (int r = 0; r < PER; ++r) e[r] = entry[warp * (32 * PER) + r * 32 + lane];
  }
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const long long n = n0 + r * 32;
    if (n < p.N) {
      p.key_out[n] = e[r].x;
      p.pos_out[n] = e[r].y;
    }
  }
  cluster_sync_all();  // no CTA leaves while its shared memory may be written
}

// ------------------------------------------------------------------- the sums
// The sorted entries in pieces of kPiece: CTA (piece, columns) adds the rows of
// each run of equal ids.  A run inside the piece is written at once.  A run that
// began in an earlier piece leaves its part in head[piece], one that goes on
// into the next leaves the part from its beginning in tail[piece]; those parts
// are joined in order by embed_join_kernel.
constexpr int kPiece = 32;
constexpr int kSumThreads = 128;

struct EmbSumParams {
  const uint32_t* key;
  const uint32_t* pos;
  const void* dout;  // [N, D]
  void* dw;          // [V, D], zeroed
  float* head;       // [pieces, D]
  float* tail;       // [pieces, D]
  long long N;
  uint32_t V;
  int D;
  float scale;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads) embed_sum_kernel(EmbSumParams p) {
  constexpr int kBatch = 8;
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t key[kPiece + 2], pos[kPiece];  // key[0]: the entry before, key[cnt + 1]: after
  const long long e0 = (long long)blockIdx.x * kPiece;
  const int cnt = int(min((long long)kPiece, p.N - e0));
  for (int i = threadIdx.x; i < cnt + 2; i += kSumThreads) {
    const long long e = e0 + i - 1;
    key[i] = e >= 0 && e < p.N ? p.key[e] : 0xffffffffu;
    if (i >= 1 && i <= cnt) pos[i - 1] = p.pos[e];
  }
  __syncthreads();
  const int c = (blockIdx.y * kSumThreads + threadIdx.x) * VEC;
  if (c >= p.D) return;
  const T* src = static_cast<const T*>(p.dout) + c;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  bool opened = key[0] == key[1];  // the current run began in an earlier piece
  // rows in batches, a batch's loads ahead of its sums; rows that do not count are read
  // as well, since a condition at each load makes the loads wait for one another (16384
  // tokens of 1024 bf16: 24 us against 9)
  for (int i0 = 0; i0 < cnt && key[i0 + 1] < p.V; i0 += kBatch) {
    float f[kBatch][VEC];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      EmbVec<T, VEC>::load(src + (size_t)pos[min(i0 + b, cnt - 1)] * p.D, f[b]);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b;
      if (i >= cnt) break;
      const uint32_t v = key[i + 1];
      if (v >= p.V) break;  // the dropped entries: nothing after them counts
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += f[b][k];
      const bool goes_on = key[i + 2] == v;
      if (goes_on && i + 1 < cnt) continue;
      if (opened || goes_on) {
        float* d = (opened ? p.head : p.tail) + (size_t)blockIdx.x * p.D + c;
        if (VEC % 4 == 0) {  // D is a multiple of VEC
#pragma unroll
          for (int k = 0; k + 3 < VEC; k += 4)
            *reinterpret_cast<float4*>(d + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) d[k] = acc[k];
        }
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] *= p.scale;
        EmbVec<T, VEC>::store(static_cast<T*>(p.dw) + (size_t)v * p.D + c, acc);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
      opened = false;
    }
  }
}

// CTA (piece, 32 VEC columns at a time): if a run begins in the piece and goes on,
// the run's parts: tail[piece], then head of the pieces up to its end, in 8
// stretches side by side that are added in order.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(EmbSumParams p) {
  __shared__ float sum[8][32 * VEC];
  pdl_wait();
  pdl_trigger();
  const long long b = blockIdx.x;
  const long long last = b * kPiece + kPiece - 1;  // the piece's last entry
  if (last + 1 >= p.N) return;
  const uint32_t v = p.key[last], next = p.key[last + 1], first = p.key[b * kPiece];
  const uint32_t prev = b > 0 ? p.key[b * kPiece - 1] : 0xffffffffu;
  if (v >= p.V || next != v) return;
  if (first == v && prev == v) return;  // began earlier
  // the pieces whose first entry is of the run follow this one: the first that is not
  // among 32 at a time, a stride apart, the stride 1 at first (most runs end there)
  const int lane = threadIdx.x & 31;
  const long long pieces = (p.N + kPiece - 1) / kPiece;
  auto in_run = [&](long long q) { return q < pieces && p.key[q * kPiece] == v; };
  long long lo = b + 1, hi = pieces;  // lo: of the run, hi: not
  int cnt = __popc(__ballot_sync(0xffffffffu, in_run(lo + 1 + lane)));
  if (cnt < 32) {
    lo += cnt;
  } else {
    lo += 32;
    while (hi - lo > 1) {
      const long long step = (hi - lo + 31) / 32;
      const long long q = lo + 1 + lane * step;
      cnt = __popc(__ballot_sync(0xffffffffu, q < hi && in_run(q)));
      const long long top = lo + 1 + cnt * step;
      if (cnt) lo += 1 + (cnt - 1) * step;
      hi = top < hi ? top : hi;
    }
  }
  const long long parts = lo - b, per = (parts + 7) / 8;  // head pieces
  const int col = (threadIdx.x & 31) * VEC, g = threadIdx.x >> 5;
  for (int c0 = blockIdx.y * 32 * VEC; c0 < p.D; c0 += gridDim.y * 32 * VEC) {
    const int c = c0 + col;
    float acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    if (c < p.D) {
      if (g == 0) EmbVec<float, VEC>::load(p.tail + (size_t)b * p.D + c, acc);
      const long long e = min(parts, (g + 1) * per);
#pragma unroll 4
      for (long long q = g * per; q < e; ++q) {
        float f[VEC];
        EmbVec<float, VEC>::load(p.head + (size_t)(b + 1 + q) * p.D + c, f);
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += f[k];
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum[g][col + k] = acc[k];
    __syncthreads();
    if (g == 0 && c < p.D) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
#pragma unroll
        for (int j = 1; j < 8; ++j) acc[k] += sum[j][col + k];
        static_cast<T*>(p.dw)[(size_t)v * p.D + c + k] = T(acc[k] * p.scale);
      }
    }
    __syncthreads();
  }
}

static size_t embed_align(size_t n) { return (n + 255) / 256 * 256; }

struct EmbWork {
  uint32_t *key[2], *pos[2], *count;
  float *head, *tail;
  size_t bytes;
  EmbWork(void* base, long long N, int D) {
    const size_t tiles = size_t((N + kSortTile - 1) / kSortTile);
    const size_t pieces = size_t((N + kPiece - 1) / kPiece);
    size_t at = 0;
    auto take = [&](size_t n) {
      char* q = static_cast<char*>(base) + at;
      at += embed_align(n);
      return q;
    };
    for (int i = 0; i < 2; ++i) {
      key[i] = reinterpret_cast<uint32_t*>(take(size_t(N) * 4));
      pos[i] = reinterpret_cast<uint32_t*>(take(size_t(N) * 4));
    }
    count = reinterpret_cast<uint32_t*>(take(tiles * 256 * 4));
    head = reinterpret_cast<float*>(take(pieces * D * 4));
    tail = reinterpret_cast<float*>(take(pieces * D * 4));
    bytes = at;
  }
};

static int embed_vec(int D, int es, const void* a, const void* b) {
  int vec = 16 / es;
  while (vec > 1 && (D % vec || !aligned(a, size_t(vec) * es) || !aligned(b, size_t(vec) * es)))
    vec /= 2;
  return vec;
}

static int embed_checks(int dtype, long long N, long long V, int D) {
  CYFA_REQUIRE(N > 0 && N < (1ll << 31) && V > 0 && V < (1ll << 31) && D > 0, kBadShape);
  CYFA_REQUIRE(dtype == 0 || dtype == 1, kBadDtype);
  return kOk;
}

}  // namespace cyfa

extern "C" {

int cyfa_embed_fwd(const long long* tokens, const void* weight, int dtype, void* out, long long N,
                   long long V, int D, float scale, void* stream) {
  CYFA_REQUIRE(tokens && weight && out, kNullPointer);
  const int rc = embed_checks(dtype, N, V, D);
  if (rc) return rc;
  const int es = dtype == 1 ? 2 : 4;
  CYFA_REQUIRE(aligned(tokens, 8) && aligned(weight, es) && aligned(out, es), kMisaligned);
  const int vec = embed_vec(D, es, weight, out);
  const int per_row = D / vec, per_thread = vec >= 4 ? 4 : 8;
  // Rows kernel: where a row fills half of a warp's accesses or more (16384 rows of 512
  // bf16: 12 us against 14, 65536 of 129 f32: 18 against 28; below, 65536 of 256 bf16:
  // 24 against 19).
  const bool by_rows = per_row * 2 >= per_thread * 32;
  const int parts = (per_row + per_thread * 32 - 1) / (per_thread * 32);  // warps of a row
  const long long n = by_rows ? N * parts : N * per_row;  // warps, or accesses
  const long long per_cta = by_rows ? kEmbThreads / 32 : per_thread * kEmbThreads;
  CYFA_REQUIRE((n + per_cta - 1) / per_cta < (1ll << 31), kBadShape);
  const unsigned grid = unsigned((n + per_cta - 1) / per_cta);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define CYFA_EMB(T, VEC)                                                                        \
  do {                                                                                          \
    const T* w = static_cast<const T*>(weight);                                                 \
    T* o = static_cast<T*>(out);                                                                \
    if (by_rows)                                                                                \
      CYFA_LAUNCH("embed_fwd", s, (launch_k(embed_fwd_rows_kernel<T, VEC>, grid, kEmbThreads, 0, \
                                            s, tokens, w, o, N, V, D, scale, parts)));          \
    else                                                                                        \
      CYFA_LAUNCH("embed_fwd", s, (launch_k(embed_fwd_kernel<T, VEC>, grid, kEmbThreads, 0, s,  \
                                            tokens, w, o, N, V, D, scale)));                    \
  } while (0)
  if (dtype == 1) {
    if (vec == 8) CYFA_EMB(__nv_bfloat16, 8);
    else if (vec == 4) CYFA_EMB(__nv_bfloat16, 4);
    else if (vec == 2) CYFA_EMB(__nv_bfloat16, 2);
    else CYFA_EMB(__nv_bfloat16, 1);
  } else {
    if (vec == 4) CYFA_EMB(float, 4);
    else if (vec == 2) CYFA_EMB(float, 2);
    else CYFA_EMB(float, 1);
  }
#undef CYFA_EMB
  return launch_status();
}

size_t cyfa_embed_bwd_work_bytes(long long N, int D) {
  return N > 0 && D > 0 ? EmbWork(nullptr, N, D).bytes : 0;
}

int cyfa_embed_bwd(const long long* tokens, const void* dout, int dtype, void* dweight, long long N,
                   long long V, int D, float scale, long long padding_idx, void* work,
                   size_t work_bytes, void* stream) {
  CYFA_REQUIRE(tokens && dout && dweight && work, kNullPointer);
  const int rc = embed_checks(dtype, N, V, D);
  if (rc) return rc;
  const int es = dtype == 1 ? 2 : 4;
  CYFA_REQUIRE(aligned(tokens, 8) && aligned(dout, es) && aligned(dweight, es) && aligned(work, 256),
               kMisaligned);
  const EmbWork w(work, N, D);
  CYFA_REQUIRE(work_bytes >= w.bytes, kWorkspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int cur = 0;
  if (N <= kCsMax) {
    ClusterSortParams p{};
    p.tokens = tokens;
    p.key_out = w.key[0];
    p.pos_out = w.pos[0];
    p.N = N;
    p.V = V;
    p.pad = padding_idx;
    int bits = 1;  // of the largest key, V
    while ((V >> bits) > 0) ++bits;
    p.passes = (bits + 8) / 9;
    p.bits = (bits + p.passes - 1) / p.passes;
    uint8_t* d = static_cast<uint8_t*>(dweight);
    const size_t nbytes = size_t(V) * D * es;
    const size_t lead = std::min(nbytes, (16 - reinterpret_cast<uintptr_t>(d) % 16) % 16);
    p.edge0 = d;
    p.edge0_bytes = int(lead);
    p.clear = reinterpret_cast<uint4*>(d + lead);
    p.clear_vecs = (long long)((nbytes - lead) / 16);
    p.edge1 = d + lead + p.clear_vecs * 16;
    p.edge1_bytes = int(nbytes - lead - p.clear_vecs * 16);
    // 128 KiB a clearing CTA at least, up to 128 clusters: only 16 clusters run at a
    // time, so that few large shares leave a second round (100003 x 1001 f32, 400 MB:
    // 109 us in 16 clusters, 86 in 32, 74 in 64, 71 in 128; 32000 x 1024 bf16 25, 22, 20, 23)
    const unsigned clear = unsigned(std::min<long long>(128, 1 + p.clear_vecs / (kCsCtas * 4 * kCsClear)));
    const dim3 grid(kCsCtas * (1 + clear));
#define CYFA_CS(PER)                                                                             \
  do {                                                                                           \
    set_smem(embed_cluster_sort_kernel<PER>, cs_smem<PER>());                                    \
    CYFA_LAUNCH("embed_sort", s, (launch_cluster_k(embed_cluster_sort_kernel<PER>, grid,         \
                                                   kCsThreads, kCsCtas, cs_smem<PER>(), s, p))); \
  } while (0)
    const long long per = (N + kCsCtas * kCsThreads - 1) / (kCsCtas * kCsThreads);
    if (per <= 1) CYFA_CS(1);
    else if (per <= 2) CYFA_CS(2);
    else if (per <= 4) CYFA_CS(4);
    else if (per <= 8) CYFA_CS(8);
    else CYFA_CS(16);
#undef CYFA_CS
  } else {
    const cudaError_t e = cudaMemsetAsync(dweight, 0, size_t(V) * D * es, s);
    if (e != cudaSuccess) return -static_cast<int>(e);
    SortPass p{tokens, nullptr, nullptr, w.key[0], w.pos[0], w.count, N, V, padding_idx, 0,
               int((N + kSortTile - 1) / kSortTile)};
    for (int shift = 0; shift < 32 && (V >> shift) > 0; shift += 8) {
      p.shift = shift;
      CYFA_LAUNCH("embed_sort_count", s,
                  (launch_k(embed_sort_count_kernel, unsigned(p.tiles), kSortThreads, 0, s, p)));
      CYFA_LAUNCH("embed_sort_scan", s,
                  (launch_k(embed_sort_scan_kernel, 1, 1024, 0, s, w.count, p.tiles * 256)));
      CYFA_LAUNCH("embed_sort_move", s,
                  (launch_k(embed_sort_move_kernel, unsigned(p.tiles), kSortThreads, 0, s, p)));
      cur = p.key_out == w.key[0] ? 0 : 1;
      p.tokens = nullptr;
      p.key_in = w.key[cur];
      p.pos_in = w.pos[cur];
      p.key_out = w.key[1 - cur];
      p.pos_out = w.pos[1 - cur];
    }
  }
  EmbSumParams q{w.key[cur], w.pos[cur], dout, dweight, w.head, w.tail, N, uint32_t(V), D, scale};
  const int vec = embed_vec(D, es, dout, dweight);
  const unsigned pieces = unsigned((N + kPiece - 1) / kPiece);
  const int cols = kSumThreads * vec;
  CYFA_REQUIRE((D + cols - 1) / cols <= 65535, kBadShape);
  const dim3 grid(pieces, unsigned((D + cols - 1) / cols));
#define CYFA_EMB(T, VEC) \
  CYFA_LAUNCH("embed_sum", s, (launch_k(embed_sum_kernel<T, VEC>, grid, kSumThreads, 0, s, q)))
  if (dtype == 1) {
    if (vec == 8) CYFA_EMB(__nv_bfloat16, 8);
    else if (vec == 4) CYFA_EMB(__nv_bfloat16, 4);
    else if (vec == 2) CYFA_EMB(__nv_bfloat16, 2);
    else CYFA_EMB(__nv_bfloat16, 1);
  } else {
    if (vec == 4) CYFA_EMB(float, 4);
    else if (vec == 2) CYFA_EMB(float, 2);
    else CYFA_EMB(float, 1);
  }
#undef CYFA_EMB
  if (pieces > 1) {
    // (a partial row starts at a multiple of 4 bytes D: float4 where D allows it)
    const int jcols = D % 4 == 0 ? 128 : 32;
    const dim3 jgrid(pieces - 1, unsigned(std::min((D + jcols - 1) / jcols, 8)));
#define CYFA_EMB_JOIN(T, VEC) \
  CYFA_LAUNCH("embed_join", s, (launch_k(embed_join_kernel<T, VEC>, jgrid, 256, 0, s, q)))
    if (dtype == 1) {
      if (D % 4 == 0) CYFA_EMB_JOIN(__nv_bfloat16, 4); else CYFA_EMB_JOIN(__nv_bfloat16, 1);
    } else {
      if (D % 4 == 0) CYFA_EMB_JOIN(float, 4); else CYFA_EMB_JOIN(float, 1);
    }
#undef CYFA_EMB_JOIN
  }
  return launch_status();
}

}  // extern "C"
