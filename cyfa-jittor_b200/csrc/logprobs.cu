// Log probabilities of given tokens from a row of logits x [V], with the
// distribution's entropy and its most likely alternatives, and the gradient of
// the first two.
//   m = max x,  s = sum e^(x - m),  t = sum (x - m) e^(x - m)
//   log p_j = (x_j - m) - log s,    H = -sum p log p = log s - t / s
//   d/dx_j (g log p_id + h H) = g [j = id] - p_j (g + h (log p_j + H))
// One pass over the row keeps (m, s, t) per thread, all in fp32, and rescales
// the sums when a larger maximum arrives.  Masked entries (-inf) have p = 0 and
// add nothing; a row with no finite entry has log p = -inf, H = 0 and zero
// gradient; NaN or +inf in a row makes its log p and H NaN.
//
// Alternatives are ordered by (logit, then lowest index), as the 64-bit key
// ordered(x) << 32 | ~index.  The k-th largest of the thread groups' maxima is a
// lower bound of the k-th largest key, so a second read of the row (from cache)
// collects the few keys above it, which are ranked by counting.
#include "cyfa_common.cuh"

namespace cyfa {

constexpr int kLpThreads = 512;
constexpr int kLpGroups = 128;   // lanes of one group: kLpThreads / kLpGroups
constexpr int kLpMaxTop = 32;    // <= kLpGroups
constexpr int kLpCand = 1024;    // candidates kept before the slow path takes over

struct LogprobParams {
  const void* x;
  long long inner, s_outer, s_inner;  // row r: x + (r / inner) s_outer + (r % inner) s_inner
  const long long* tokens;            // [rows]
  long long ignore;
  float* logp;              // [rows]
  float* entropy;           // [rows]
  float2* stats;            // [rows] (m, log s), may be null forward
  float* top_logp;          // [rows, top]
  long long* top_tokens;    // [rows, top]
  int V, top;
  // backward
  const float* dlogp;       // [rows] or null
  const float* dentropy;    // [rows] or null
  void* dx;                 // [rows, V] contiguous
  int nseg;                 // CTAs of one row
};

template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <>
struct LpVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) { unpack_bf16x8(u, f); }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]),
                      pack_bf16(f[6], f[7]));
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) {
    return __bfloat162float(*p);
  }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) {
    *p = __float2bfloat16_rn(v);
  }
};

// Unsigned order of floats: -inf lowest, -0 equal to +0, NaN above +inf.
__device__ __forceinline__ uint32_t lp_order(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = x == 0.f ? 0u : __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_unorder(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long lp_key(float x, int idx) {
  return (static_cast<unsigned long long>(lp_order(x)) << 32) | static_cast<uint32_t>(~idx);
}

struct LpSums {
  float m, s, t;
};
// e^(x - m) and its product with x - m; m finite.  x - m is formed before the
// scaling to base 2 so that nearby values keep their digits, and clamped for the
// product only: e is 0 there, and NaN stays NaN through e.
__device__ __forceinline__ void lp_term(float x, float m, float& s, float& t) {
  const float d = x - m;
  const float e = fast_exp2(d * kLog2e);
  s += e;
  t = fmaf(fmaxf(d, -1e25f), e, t);
}
__device__ __forceinline__ LpSums lp_merge(LpSums a, LpSums b) {
  LpSums r;
  r.m = fmaxf(a.m, b.m);
  const float base = r.m == -INFINITY ? 0.f : r.m;
  // a side without finite entries has m = -inf and s = t = 0 (or NaN to pass on)
  const float da = fmaxf(a.m - base, -1e25f), db = fmaxf(b.m - base, -1e25f);
  const float ea = fast_exp2(da * kLog2e), eb = fast_exp2(db * kLog2e);
  r.s = a.s * ea + b.s * eb;
  r.t = fmaf(da, a.s, a.t) * ea + fmaf(db, b.s, b.t) * eb;
  return r;
}
__device__ __forceinline__ LpSums lp_shfl(LpSums a, int o) {
  LpSums b;
  b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
  b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
  b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
  return b;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_map(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ float cluster_ld_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long cluster_ld_u64(uint32_t a) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

// The n elements of a row part starting at p: `head` elements up to the first
// 16-byte boundary, nvec vectors, then the rest.
template <typename T>
struct LpSpan {
  const T* p;
  int n, head, nvec;
  __device__ __forceinline__ LpSpan(const T* p_, int n_) : p(p_), n(n_) {
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / int(sizeof(T));
    head = min(n, mis ? LpVec<T>::N - mis : 0);
    nvec = (n - head) / LpVec<T>::N;
  }
  __device__ __forceinline__ int loose() const { return n - nvec * LpVec<T>::N; }  // head + tail
  __device__ __forceinline__ int loose_index(int i) const {
    return i < head ? i : i + nvec * LpVec<T>::N;
  }
};

// One row per cluster; the cluster's CTAs split the row.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprob_fwd_kernel(LogprobParams p) {
  constexpr int N = LpVec<T>::N, kUnroll = 4;
  constexpr int kLanes = kLpThreads / kLpGroups, kWarps = kLpThreads / 32;
  __shared__ LpSums s_warp[kWarps];
  __shared__ LpSums s_part;                            // this CTA's sums
  __shared__ unsigned long long s_group[kLpGroups];
  __shared__ unsigned long long s_cand[kLpCand];
  __shared__ unsigned long long s_best[kLpMaxTop];     // this CTA's k largest keys
  __shared__ unsigned long long s_bound;
  __shared__ int s_count;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), csize = cluster_size();
  const long long row = blockIdx.x / csize;
  const T* xr = static_cast<const T*>(p.x) + (row / p.inner) * p.s_outer + (row % p.inner) * p.s_inner;
  const int seg = ((p.V + int(csize) - 1) / int(csize) + 63) / 64 * 64;
  const int j0 = min(p.V, int(rank) * seg), n = min(p.V, j0 + seg) - j0;
  const LpSpan<T> sp(xr + j0, n);
  const uint4* body = reinterpret_cast<const uint4*>(sp.p + sp.head);

  LpSums a{-INFINITY, 0.f, 0.f};
  int at = -1;  // index of the thread's first largest entry (its first entry at the start)
  if (tid < sp.loose()) {
    at = sp.loose_index(tid);
    const float x = LpVec<T>::get(sp.p + at);
    a.m = fmaxf(a.m, x);
    lp_term(x, a.m == -INFINITY ? 0.f : a.m, a.s, a.t);
  }
  for (int v0 = tid; v0 < sp.nvec; v0 += kLpThreads * kUnroll) {
    uint4 u[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (v0 + k * kLpThreads < sp.nvec) u[k] = body[v0 + k * kLpThreads];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int v = v0 + k * kLpThreads;
      if (v < sp.nvec) {
        float f[N];
        LpVec<T>::unpack(u[k], f);
        float bm = f[0];
#pragma unroll
        for (int i = 1; i < N; ++i) bm = fmaxf(bm, f[i]);
        if (at < 0) at = sp.head + v * N;
        if (bm > a.m) {
          if (p.top) {
#pragma unroll
            for (int i = N - 1; i >= 0; --i)
              if (f[i] == bm) at = sp.head + v * N + i;
          }
          a = lp_merge(a, LpSums{bm, 0.f, 0.f});
        }
        const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
        for (int i = 0; i < N; ++i) lp_term(f[i], base, a.s, a.t);
      }
    }
  }
  // key of the thread's largest entry (a lower bound of it if that is NaN)
  unsigned long long best = at < 0 ? 0ull : lp_key(a.m, j0 + at);
#pragma unroll
  for (int o = 16; o; o >>= 1) a = lp_merge(a, lp_shfl(a, o));
  if (lane == 0) s_warp[warp] = a;
  if (p.top) {
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) {
      const unsigned long long b = __shfl_xor_sync(0xffffffffu, best, o);
      best = b > best ? b : best;
    }
    if (tid % kLanes == 0) s_group[tid / kLanes] = best;
    if (tid == 0) {
      s_count = 0;
      s_bound = 0;
    }
    if (tid < kLpMaxTop) s_best[tid] = 0;
  }
  __syncthreads();
  if (warp == 0) {
    a = lane < kWarps ? s_warp[lane] : LpSums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o; o >>= 1) a = lp_merge(a, lp_shfl(a, o));
    if (lane == 0) s_part = a;
  }
  if (p.top) {
    const int top = min(p.top, n);  // of this part
    if (tid < kLpGroups && top > 0) {
      const unsigned long long mine = s_group[tid];
      int above = 0, same = 0;
      for (int i = 0; i < kLpGroups; ++i) {
        above += s_group[i] > mine;
        same += s_group[i] == mine;  // empty groups share the key 0
      }
      if (above < top && above + same >= top) s_bound = mine;
    }
    __syncthreads();
    if (top > 0) {
      const unsigned long long bound = s_bound;
      const float low = lp_unorder(static_cast<uint32_t>(bound >> 32));
      auto offer = [&](float x, int j) {
        if (bound != 0 && x < low) return;
        const unsigned long long key = lp_key(x, j0 + j);
        if (key < bound) return;
        const int c = atomicAdd(&s_count, 1);
        if (c < kLpCand) s_cand[c] = key;
      };
      if (tid < sp.loose()) {
        const int j = sp.loose_index(tid);
        offer(LpVec<T>::get(sp.p + j), j);
      }
      for (int v = tid; v < sp.nvec; v += kLpThreads) {
        float f[N];
        LpVec<T>::unpack(body[v], f);
#pragma unroll
        for (int i = 0; i < N; ++i) offer(f[i], sp.head + v * N + i);
      }
      __syncthreads();
      const int cnt = s_count;
      if (cnt <= kLpCand) {
        for (int c = tid; c < cnt; c += kLpThreads) {
          const unsigned long long mine = s_cand[c];
          int above = 0;
          for (int i = 0; i < cnt; ++i) above += s_cand[i] > mine;
          if (above < top) s_best[above] = mine;
        }
      } else {
        // more keys above the bound than are kept (they sit in fewer than k
        // groups): one maximum below the last at a time
        unsigned long long last = ~0ull;
        for (int k = 0; k < top; ++k) {
          unsigned long long b = 0;
          for (int j = tid; j < n; j += kLpThreads) {
            const unsigned long long key = lp_key(LpVec<T>::get(sp.p + j), j0 + j);
            if (key < last && key > b) b = key;
          }
#pragma unroll
          for (int o = 16; o; o >>= 1) {
            const unsigned long long c = __shfl_xor_sync(0xffffffffu, b, o);
            b = c > b ? c : b;
          }
          __syncthreads();
          if (lane == 0) s_group[warp] = b;
          __syncthreads();
          b = s_group[0];
          for (int w = 1; w < kWarps; ++w) b = s_group[w] > b ? s_group[w] : b;
          last = b;
          if (tid == 0) s_best[k] = b;
        }
      }
    }
  }
  if (csize > 1) {
    cluster_sync_all();
  } else {
    __syncthreads();
  }
  if (rank == 0) {
    LpSums tot = s_part;
    for (uint32_t c = 1; c < csize; ++c) {
      const uint32_t at_c = cluster_map(smem_u32(&s_part), c);
      tot = lp_merge(tot, LpSums{cluster_ld_f32(at_c), cluster_ld_f32(at_c + 4),
                                 cluster_ld_f32(at_c + 8)});
    }
    const bool empty = tot.m == -INFINITY && tot.s == 0.f;
    const float logs = empty ? 0.f : logf(tot.s);
    if (tid == 0) {
      const float h = empty ? 0.f : logs - tot.t / tot.s;
      p.entropy[row] = h < 0.f ? 0.f : h;
      if (p.stats) p.stats[row] = make_float2(tot.m, logs);
      const long long id = p.tokens[row];
      float lp = 0.f;
      if (id != p.ignore) {
        if (id < 0 || id >= p.V) {
          set_error(kErrBadIndex);
          lp = __uint_as_float(0x7fffffffu);
        } else {
          lp = empty ? -INFINITY : (LpVec<T>::get(xr + id) - tot.m) - logs;
        }
      }
      p.logp[row] = lp;
    }
    if (p.top) {
      // the cluster's best keys, ranked by counting
      const int total = int(csize) * p.top;
      for (int c = tid; c < total; c += kLpThreads)
        s_cand[c] = csize == 1 ? s_best[c]
                               : cluster_ld_u64(cluster_map(smem_u32(&s_best[c % p.top]), c / p.top));
      __syncthreads();
      for (int c = tid; c < total; c += kLpThreads) {
        const unsigned long long mine = s_cand[c];
        if (mine == 0) continue;  // a part shorter than k
        int above = 0;
        for (int i = 0; i < total; ++i) above += s_cand[i] > mine;
        if (above < p.top) {
          const float x = lp_unorder(static_cast<uint32_t>(mine >> 32));
          const int j = static_cast<int>(~static_cast<uint32_t>(mine));
          p.top_tokens[row * p.top + above] = j;
          p.top_logp[row * p.top + above] = empty ? -INFINITY : (x - tot.m) - logs;
        }
      }
    }
  }
  if (csize > 1) cluster_sync_all();  // no CTA leaves while its shared memory is read
}

constexpr int kLpBwdThreads = 256;
constexpr int kLpBwdVecs = 4;  // vectors of a thread

// CTA (row, segment): reads its logits once, writes their gradient.  VECTOR:
// input and output rows are misaligned alike, so both use 16-byte accesses
// after the same head; otherwise element accesses.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kLpBwdThreads) logprob_bwd_kernel(LogprobParams p) {
  constexpr int N = LpVec<T>::N, kSpan = kLpBwdThreads * kLpBwdVecs * N;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / p.nseg;
  const int part = int(blockIdx.x % p.nseg);
  const T* xr = static_cast<const T*>(p.x) + (row / p.inner) * p.s_outer + (row % p.inner) * p.s_inner;
  T* dr = static_cast<T*>(p.dx) + row * p.V;
  const LpSpan<T> sp(xr, p.V);
  const uint4* src = reinterpret_cast<const uint4*>(xr + sp.head);
  uint4* dst = reinterpret_cast<uint4*>(dr + sp.head);
  uint4 u[kLpBwdVecs];
  const int v0 = part * kLpBwdThreads * kLpBwdVecs + tid;
  if (VECTOR) {
#pragma unroll
    for (int k = 0; k < kLpBwdVecs; ++k)
      if (v0 + k * kLpBwdThreads < sp.nvec) u[k] = __ldcs(src + v0 + k * kLpBwdThreads);
  }
  const float2 st = p.stats[row];
  const float H = p.entropy[row];
  const long long id = p.tokens[row];
  const bool live = id >= 0 && id < p.V && id != p.ignore;
  const float g = live && p.dlogp ? p.dlogp[row] : 0.f;
  const float h = p.dentropy ? p.dentropy[row] : 0.f;
  // p_j (g + h (lp_j + H)) = p_j (h lp_j + c)
  const float base = st.x == -INFINITY ? 0.f : st.x, c = fmaf(h, H, g);
  auto grad = [&](float x, int j) {
    const float lp = (x - base) - st.y;
    const float pj = fast_exp2(lp * kLog2e);
    const float d = -pj * fmaf(h, fmaxf(lp, -1e25f), c);
    return j == id && live ? d + g : d;
  };
  if (VECTOR) {
#pragma unroll
    for (int k = 0; k < kLpBwdVecs; ++k) {
      const int v = v0 + k * kLpBwdThreads;
      if (v < sp.nvec) {
        float f[N];
        LpVec<T>::unpack(u[k], f);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = grad(f[i], sp.head + v * N + i);
        __stcs(dst + v, LpVec<T>::pack(f));
      }
    }
    if (part == 0 && tid < sp.loose()) {
      const int j = sp.loose_index(tid);
      LpVec<T>::put(dr + j, grad(LpVec<T>::get(xr + j), j));
    }
  } else {
    const int end = min((long long)p.V, (long long)(part + 1) * kSpan);
    for (int j = part * kSpan + tid; j < end; j += kLpBwdThreads)
      LpVec<T>::put(dr + j, grad(LpVec<T>::get(xr + j), j));
  }
}

}  // namespace cyfa

using namespace cyfa;

namespace cyfa {

template <typename... KArgs, typename... Args>
static void launch_cluster_k(void (*kernel)(KArgs...), dim3 grid, dim3 block, unsigned cluster,
                             size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = g_pdl.load(std::memory_order_relaxed);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

static int logprob_checks(const void* logits, int dtype, long long rows, long long inner,
                          long long s_outer, long long s_inner, int V) {
  CYFA_REQUIRE(rows > 0 && inner > 0 && s_outer >= 0 && s_inner >= 0 && V > 0 && V < (1 << 30), kBadShape);
  CYFA_REQUIRE(dtype == 0 || dtype == 1, kBadDtype);
  CYFA_REQUIRE(aligned(logits, dtype == 1 ? 2 : 4), kMisaligned);
  return kOk;
}

}  // namespace cyfa

extern "C" {

int cyfa_token_logprobs_fwd(const void* logits, int dtype, long long rows, long long inner,
                            long long stride_outer, long long stride_inner, int V,
                            const long long* tokens, long long ignore_index, int top, float* logp,
                            float* entropy, float* stats, float* top_logp, long long* top_tokens,
                            void* stream) {
  CYFA_REQUIRE(logits && tokens && logp && entropy && (top == 0 || (top_logp && top_tokens)),
               kNullPointer);
  const int rc = logprob_checks(logits, dtype, rows, inner, stride_outer, stride_inner, V);
  if (rc) return rc;
  CYFA_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= V && rows < (1ll << 27), kBadShape);
  CYFA_REQUIRE(aligned(tokens, 8) && (!stats || aligned(stats, 8)) && aligned(logp, 4) && aligned(entropy, 4) &&
                   (!top || (aligned(top_logp, 4) && aligned(top_tokens, 8))),
               kMisaligned);
  LogprobParams p{};
  p.x = logits;
  p.inner = inner;
  p.s_outer = stride_outer;
  p.s_inner = stride_inner;
  p.tokens = tokens;
  p.ignore = ignore_index;
  p.logp = logp;
  p.entropy = entropy;
  p.stats = reinterpret_cast<float2*>(stats);
  p.top_logp = top_logp;
  p.top_tokens = top_tokens;
  p.V = V;
  p.top = top;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  unsigned cluster = 1;
  while (cluster < 8 && rows * cluster < 296 && V / int(cluster) > 4096) cluster *= 2;
  const dim3 grid(unsigned(rows * cluster));
  if (dtype == 1)
    CYFA_LAUNCH("logprob_fwd", s, (launch_cluster_k(logprob_fwd_kernel<__nv_bfloat16>, grid,
                                                    kLpThreads, cluster, 0, s, p)));
  else
    CYFA_LAUNCH("logprob_fwd", s, (launch_cluster_k(logprob_fwd_kernel<float>, grid, kLpThreads,
                                                    cluster, 0, s, p)));
  return launch_status();
}

int cyfa_token_logprobs_bwd(const void* logits, int dtype, long long rows, long long inner,
                            long long stride_outer, long long stride_inner, int V,
                            const long long* tokens, long long ignore_index, const float* stats,
                            const float* entropy, const float* dlogp, const float* dentropy,
                            void* dlogits, void* stream) {
  CYFA_REQUIRE(logits && tokens && stats && entropy && dlogits, kNullPointer);
  const int rc = logprob_checks(logits, dtype, rows, inner, stride_outer, stride_inner, V);
  if (rc) return rc;
  const int es = dtype == 1 ? 2 : 4;
  CYFA_REQUIRE(aligned(tokens, 8) && aligned(stats, 8) && aligned(entropy, 4) && aligned(dlogits, es) &&
                   (!dlogp || aligned(dlogp, 4)) && (!dentropy || aligned(dentropy, 4)),
               kMisaligned);
  const int span = kLpBwdThreads * kLpBwdVecs * (16 / es);
  const long long nseg = (V + span - 1) / span;
  CYFA_REQUIRE(rows * nseg < (1ll << 31), kBadShape);
  LogprobParams p{};
  p.x = logits;
  p.inner = inner;
  p.s_outer = stride_outer;
  p.s_inner = stride_inner;
  p.tokens = tokens;
  p.ignore = ignore_index;
  p.entropy = const_cast<float*>(entropy);
  p.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  p.V = V;
  p.dlogp = dlogp;
  p.dentropy = dentropy;
  p.dx = dlogits;
  p.nseg = int(nseg);
  // every row misaligned alike in input and output: bases congruent, and either
  // level's stride congruent to the dense one wherever that level is stepped
  const long long dense = (long long)V * es;
  const bool vector =
      (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) % 16 == 0 &&
      (inner == 1 || (stride_inner * es - dense) % 16 == 0) &&
      (rows <= inner || (stride_outer * es - dense * inner) % 16 == 0);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(unsigned(rows * nseg));
#define CYFA_LP_BWD(T, VEC) \
  CYFA_LAUNCH("logprob_bwd", s, (launch_k(logprob_bwd_kernel<T, VEC>, grid, kLpBwdThreads, 0, s, p)))
  if (dtype == 1) {
    if (vector) CYFA_LP_BWD(__nv_bfloat16, true); else CYFA_LP_BWD(__nv_bfloat16, false);
  } else {
    if (vector) CYFA_LP_BWD(float, true); else CYFA_LP_BWD(float, false);
  }
#undef CYFA_LP_BWD
  return launch_status();
}

}  // extern "C"
