// Log probabilities of given tokens from a row of logits x [V], with the
// distribution's entropy and its most likely alternatives, and the gradient of
// the first two.
//   m = max x,  s = sum e^(x - m),  t = sum (x - m) e^(x - m)
//   log p_j = (x_j - m) - log s,    H = -sum p log p = log s - t / s
//   d/dx_j (g log p_id + h H) = g [j = id] - p_j (g + h (log p_j + H))
// One pass over the row keeps (m, s, t) per thread, all in fp32, and rescales
// the sums when a larger maximum arrives.  Masked entries (-inf) have p = 0 and
// add nothing; a row with no finite entry has log p = -inf, H = 0 and p = 0 throughout,
// so that its gradient is g at id and 0 elsewhere, as at any masked id; NaN or +inf in
// a row makes its log p and H NaN.
//
// Alternatives are ordered by (logit, then lowest index), as the 64-bit key
// ordered(x) << 32 | ~index.  The k-th largest of the thread groups' maxima is a
// lower bound of the k-th largest key, so a second read of the row (from cache)
// collects the few keys above it, which are ranked by counting.
//
// Bound by memory where there is enough to read: 16384 rows of 32000 bf16 take 172 us
// forward (1.05 GB at 6.1 TB/s) and 341 us backward (2.1 GB at 6.2), 93 % of what a copy
// reaches; a thread keeps eight 16-byte loads in flight, and the entry's FMA, exponential
// and two sums fill 74 % (forward) and 90 % (backward) of the issue slots meanwhile.  One row (split over a
// cluster) takes 9 us and 256 rows with 20 alternatives 13 us: the latency of the
// launch, the two reads and the joins.
#include "cyfa_common.cuh"

namespace cyfa {

constexpr int kLpGroups = 128;   // groups of a CTA's threads with alternatives
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
  static constexpr uint32_t kMasked = 0xff800000u;  // a word of -inf
  // largest entry (of two vectors: entry by entry); NaN is passed over, or passed on
  static __device__ __forceinline__ float top(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                 fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ uint32_t top_word(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ uint4 top2(const uint4& a, const uint4& b) {
    return make_uint4(top_word(a.x, b.x), top_word(a.y, b.y), top_word(a.z, b.z), top_word(a.w, b.w));
  }
  static __device__ __forceinline__ float top_nan(const uint4& u) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)),
                   max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
  }
  // the entries, none below -1e38
  static __device__ __forceinline__ void finite(const uint4& u, float* f) {
    f[0] = max_nan(__uint_as_float(u.x), -1e38f);
    f[1] = max_nan(__uint_as_float(u.y), -1e38f);
    f[2] = max_nan(__uint_as_float(u.z), -1e38f);
    f[3] = max_nan(__uint_as_float(u.w), -1e38f);
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
  static constexpr uint32_t kMasked = 0xff80ff80u;
  static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t w) {
    return *reinterpret_cast<const __nv_bfloat162*>(&w);
  }
  static __device__ __forceinline__ uint32_t top_word(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(pair(a), pair(b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  static __device__ __forceinline__ uint4 top2(const uint4& a, const uint4& b) {
    return make_uint4(top_word(a.x, b.x), top_word(a.y, b.y), top_word(a.z, b.z), top_word(a.w, b.w));
  }
  static __device__ __forceinline__ float top(const uint4& u) {
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(pair(u.x), pair(u.y)),
                                                __hmax2(pair(u.z), pair(u.w))));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ float top_nan(const uint4& u) {
    const float2 f = __bfloat1622float2(__hmax2_nan(__hmax2_nan(pair(u.x), pair(u.y)),
                                                    __hmax2_nan(pair(u.z), pair(u.w))));
    return LpVec<float>::max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ void finite(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 0xfe96: -0.997e38
      const float2 x = __bfloat1622float2(__hmax2_nan(pair(w[i]), pair(0xfe96fe96u)));
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
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
// The sums are kept in base 2 about c = fl(m log2 e), so that an entry costs one
// FMA before its exponential: q = x log2 e - c, s = sum 2^q, t = sum q 2^q.  c's
// rounding shifts every q by off = m log2 e - c (exact by FMA, |off| < 1 for
// |c| <= 1e6), which the end takes out again; log2 e's own rounding scales x - m by
// 1 + 2^-25.  Beyond |c| = 1e6 the difference x - m is formed first and off is 0.
constexpr float kLpNear = 1e6f;  // bound of |c|
__device__ __forceinline__ float lp_off(float m) {
  return fabsf(m * kLog2e) <= kLpNear ? fmaf(m, kLog2e, -(m * kLog2e)) : 0.f;
}
// One entry, any finite m.  q is clamped in the product only: 2^q is 0 there, and
// NaN stays NaN through it.
__device__ __forceinline__ void lp_term(float x, float m, float& s, float& t) {
  const float q = fmaf(x - m, kLog2e, lp_off(m));
  const float e = fast_exp2(q);
  s += e;
  t = fmaf(fmaxf(q, -1e25f), e, t);
}
// s and t about m, moved to the larger maximum to (m = -inf: empty sums)
__device__ __forceinline__ void lp_rebase(float m, float to, float& s, float& t) {
  const float d = fmaxf(fmaf(m - to, kLog2e, lp_off(to) - (m == -INFINITY ? 0.f : lp_off(m))), -1e25f);
  const float e = fast_exp2(d);
  t = fmaf(d, s, t) * e;
  s *= e;
}
// The sums of WIDTH neighbouring lanes: the maximum first, each lane's sums moved
// to it once, then plain adds.
template <int WIDTH>
__device__ __forceinline__ LpSums lp_join(LpSums a) {
  float m = a.m;
#pragma unroll
  for (int o = WIDTH / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  lp_rebase(a.m, m == -INFINITY ? 0.f : m, a.s, a.t);
#pragma unroll
  for (int o = WIDTH / 2; o; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
  a.m = m;
  return a;
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
__device__ __forceinline__ uint32_t cluster_ld_u32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_st_u2(uint32_t a, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(v.x), "r"(v.y) : "memory");
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

template <typename T, int BATCH>
__device__ __forceinline__ float lp_batch_max(const uint4 (&u)[BATCH]) {
  uint4 m = u[0];
#pragma unroll
  for (int k = 1; k < BATCH; ++k) m = LpVec<T>::top2(m, u[k]);
  return LpVec<T>::top(m);
}

// A thread's sums, about a base that follows the largest entry so far from at most
// kLpSlack below (e^8 keeps the sums far inside fp32's range), so that most steps
// need not move them.
constexpr float kLpSlack = 8.f;
struct LpState {
  LpSums a{-INFINITY, 0.f, 0.f};  // m: the base
  float c = 0.f;                  // m log2 e
  float top = -INFINITY;          // the largest entry
  __device__ __forceinline__ void move(float to) {
    lp_rebase(a.m, to, a.s, a.t);
    a.m = to;
    c = to * kLog2e;
  }
  // sums about the largest entry
  __device__ __forceinline__ LpSums sums() {
    if (a.m != top) move(top);
    return a;
  }
};

// Adds a step's entries, of largest value bm.
template <typename T, int BATCH>
__device__ __forceinline__ void lp_batch(const uint4 (&u)[BATCH], float bm, LpState& st) {
  constexpr int N = LpVec<T>::N;
  LpSums& a = st.a;
  st.top = fmaxf(st.top, bm);
  if (bm > a.m + kLpSlack) st.move(bm);
  if (fabsf(st.c) <= kLpNear) {
    float s1 = 0.f, t1 = 0.f;  // second pair of chains
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      // masked entries as -1e38: 2^q is 0 and q finite
      float f[N];
      LpVec<T>::finite(u[k], f);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float q0 = fmaf(f[i], kLog2e, -st.c), q1 = fmaf(f[i + 1], kLog2e, -st.c);
        const float e0 = fast_exp2(q0), e1 = fast_exp2(q1);
        a.s += e0;
        s1 += e1;
        a.t = fmaf(q0, e0, a.t);
        t1 = fmaf(q1, e1, t1);
      }
    }
    a.s += s1;
    a.t += t1;
  } else {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      float f[N];
      LpVec<T>::unpack(u[k], f);
#pragma unroll
      for (int i = 0; i < N; ++i) lp_term(f[i], a.m, a.s, a.t);
    }
  }
}
__device__ __forceinline__ void lp_single(float x, LpState& st) {
  st.top = fmaxf(st.top, x);
  if (x > st.a.m + kLpSlack) st.move(x);
  lp_term(x, st.a.m == -INFINITY ? 0.f : st.a.m, st.a.s, st.a.t);
}

// The row's results from its sums.
template <typename T>
__device__ __forceinline__ LpSums lp_finish(const LogprobParams& p, long long row, const LpSums& a,
                                            long long id, float x_id) {
  const bool empty = a.m == -INFINITY && a.s == 0.f;
  // s about m itself, as 2^off is computed for the largest entry, and the mean of
  // x - m: both exact for a row of one entry, whose q is off
  const float off = empty ? 0.f : lp_off(a.m);
  const float logs = empty ? 0.f : logf(a.s / fast_exp2(off));
  float mean = a.t / a.s - off;
  if (fabsf(mean) <= 2.4e-7f * fabsf(off)) mean = 0.f;  // off's rounding in the product
  const float h = empty ? 0.f : fmaf(-0.69314718055994531f, mean, logs);
  p.entropy[row] = h < 0.f ? 0.f : h;
  if (p.stats) p.stats[row] = make_float2(a.m, logs);
  float lp = 0.f;
  if (id != p.ignore) {
    if (id < 0 || id >= p.V) {
      set_error(kErrBadIndex);
      lp = __uint_as_float(0x7fffffffu);
    } else {
      lp = empty ? -INFINITY : (x_id - a.m) - logs;
    }
  }
  p.logp[row] = lp;
  return LpSums{a.m, logs, empty ? 1.f : 0.f};
}

template <typename T>
__device__ __forceinline__ const T* lp_row(const LogprobParams& p, long long row) {
  const unsigned r = unsigned(row), n = unsigned(p.inner);  // rows < 2^27, inner <= rows
  const unsigned o = r / n;
  return static_cast<const T*>(p.x) + o * p.s_outer + (r - o * n) * p.s_inner;
}

// One row per cluster; the cluster's CTAs split the row.  A thread takes BATCH
// vectors a step.
template <typename T, bool TOP>
constexpr int lp_threads() {
  return TOP ? 256 : 128;
}
template <typename T, bool TOP>
__global__ void __launch_bounds__(lp_threads<T, TOP>()) logprob_fwd_kernel(LogprobParams p) {
  constexpr int N = LpVec<T>::N, kUnroll = TOP ? 4 : 8, kLpThreads = lp_threads<T, TOP>();
  constexpr int kLanes = TOP ? kLpThreads / kLpGroups : 1, kWarps = kLpThreads / 32;
  __shared__ LpSums s_warp[kWarps];
  __shared__ LpSums s_part;                                  // this CTA's sums
  __shared__ LpSums s_row;                                   // the row's
  __shared__ unsigned long long s_group[kLpGroups];
  __shared__ unsigned long long s_cand[TOP ? kLpCand : 1];
  __shared__ unsigned long long s_best[kLpMaxTop];           // this CTA's k largest keys
  __shared__ unsigned long long s_bound;
  __shared__ int s_count;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), csize = cluster_size();
  const long long row = blockIdx.x / csize;
  const T* xr = lp_row<T>(p, row);
  const int seg = ((p.V + int(csize) - 1) / int(csize) + 63) / 64 * 64;
  const int j0 = min(p.V, int(rank) * seg), n = min(p.V, j0 + seg) - j0;
  const LpSpan<T> sp(xr + j0, n);
  const uint4* body = reinterpret_cast<const uint4*>(sp.p + sp.head);

  LpState st;
  int at = -1;  // index of the thread's first largest entry (its first entry at the start)
  for (int v0 = tid; v0 < sp.nvec; v0 += kLpThreads * kUnroll) {
    uint4 u[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      u[k] = v0 + k * kLpThreads < sp.nvec
                 ? body[v0 + k * kLpThreads]
                 : make_uint4(LpVec<T>::kMasked, LpVec<T>::kMasked, LpVec<T>::kMasked,
                              LpVec<T>::kMasked);
    if (TOP && at < 0) at = sp.head + v0 * N;
    const float bm = lp_batch_max<T, kUnroll>(u);
    if (TOP && bm > st.top) {
#pragma unroll
      for (int k = kUnroll - 1; k >= 0; --k) {
        float f[N];
        LpVec<T>::unpack(u[k], f);
#pragma unroll
        for (int i = N - 1; i >= 0; --i)
          if (f[i] == bm) at = sp.head + (v0 + k * kLpThreads) * N + i;
      }
    }
    lp_batch<T, kUnroll>(u, bm, st);
  }
  if (tid < sp.loose()) {
    const int j = sp.loose_index(tid);
    const float x = LpVec<T>::get(sp.p + j);
    if (at < 0 || x > st.top) at = j;
    lp_single(x, st);
  }
  // key of the thread's largest entry (a lower bound of it if that is NaN)
  unsigned long long best = at < 0 ? 0ull : lp_key(st.top, j0 + at);
  LpSums a = lp_join<32>(st.sums());
  if (lane == 0) s_warp[warp] = a;
  if (TOP) {
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
    a = lp_join<kWarps>(s_warp[lane % kWarps]);
    if (lane == 0) s_part = a;
  }
  if (TOP) {
    const int top = min(p.top, n);  // of this part
    if (tid < kLpGroups && top > 0) {
      const unsigned long long mine = s_group[tid];
      int above = 0, same = 0;
#pragma unroll 8
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
      for (int v0 = tid; v0 < sp.nvec; v0 += kLpThreads * kUnroll) {
        uint4 u[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
          if (v0 + k * kLpThreads < sp.nvec) u[k] = body[v0 + k * kLpThreads];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
          const int v = v0 + k * kLpThreads;
          if (v >= sp.nvec || (bound != 0 && LpVec<T>::top_nan(u[k]) < low)) continue;
          float f[N];
          LpVec<T>::unpack(u[k], f);
#pragma unroll
          for (int i = 0; i < N; ++i) offer(f[i], sp.head + v * N + i);
        }
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
  if (csize > 1) cluster_sync_all();
  if (rank == 0) {
    if (warp == 0) {
      if (csize > 1) {
        a = LpSums{-INFINITY, 0.f, 0.f};
        if (lane < int(csize)) {
          const uint32_t at_c = cluster_map(smem_u32(&s_part), lane);
          a = LpSums{cluster_ld_f32(at_c), cluster_ld_f32(at_c + 4), cluster_ld_f32(at_c + 8)};
        }
        a = lp_join<8>(a);
      }
      if (lane == 0) {
        const long long id = p.tokens[row];
        const LpSums r = lp_finish<T>(p, row, a, id,
                                      id >= 0 && id < p.V ? LpVec<T>::get(xr + id) : 0.f);
        if (TOP) s_row = r;
      }
    }
    if (TOP) {
      // the cluster's best keys, ranked by counting
      __syncthreads();
      const int total = int(csize) * p.top;
      for (int c = tid; c < total; c += kLpThreads)
        s_cand[c] = csize == 1 ? s_best[c]
                               : cluster_ld_u64(cluster_map(smem_u32(&s_best[c % p.top]), c / p.top));
      __syncthreads();
      const LpSums r = s_row;
      for (int c = tid; c < total; c += kLpThreads) {
        const unsigned long long mine = s_cand[c];
        if (mine == 0) continue;  // a part shorter than k
        int above = 0;
        for (int i = 0; i < total; ++i) above += s_cand[i] > mine;
        if (above < p.top) {
          const float x = lp_unorder(static_cast<uint32_t>(mine >> 32));
          const int j = static_cast<int>(~static_cast<uint32_t>(mine));
          p.top_tokens[row * p.top + above] = j;
          p.top_logp[row * p.top + above] = r.t != 0.f ? -INFINITY : (x - r.m) - r.s;
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
  const T* xr = lp_row<T>(p, row);
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
    // element accesses, a batch of loads ahead of its stores
    constexpr int kBatch = kLpBwdVecs * N / 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long jb = (long long)part * kSpan + h * kBatch * kLpBwdThreads + tid;
      float f[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const long long j = jb + i * kLpBwdThreads;
        f[i] = j < p.V ? LpVec<T>::get(xr + j) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const long long j = jb + i * kLpBwdThreads;
        if (j < p.V) LpVec<T>::put(dr + j, grad(f[i], int(j)));
      }
    }
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
  CYFA_REQUIRE(rows > 0 && inner > 0 && inner <= rows && s_outer >= 0 && s_inner >= 0 && V > 0 && V < (1 << 30), kBadShape);
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
  // Rows are split while they are fewer than the SMs and stay a few thousand entries
  // (32000 bf16 entries, one row: 15.4 us unsplit, 12.0 in 8; 256 rows: 18.8 us unsplit,
  // 21.5 in 2), and where the second read of many long rows would miss the L2 cache
  // (1024 rows of 50021 f32: 87 us unsplit, 78 in 2, 97 in 4).
  const long long row_bytes = (long long)V * (dtype == 1 ? 2 : 4);
  unsigned cluster = 1;
  while (cluster < 8 && ((rows * cluster < 148 && V / int(cluster) > 4096) ||
                         (top && row_bytes / cluster > 131072)))
    cluster *= 2;
  const dim3 grid(unsigned(rows * cluster));
#define CYFA_LP_FWD(T, TOP)        \
  CYFA_LAUNCH("logprob_fwd", s,     \
              (launch_cluster_k(logprob_fwd_kernel<T, TOP>, grid, lp_threads<T, TOP>(), cluster, 0, s, p)))
  if (dtype == 1) {
    if (top) CYFA_LP_FWD(__nv_bfloat16, true); else CYFA_LP_FWD(__nv_bfloat16, false);
  } else {
    if (top) CYFA_LP_FWD(float, true); else CYFA_LP_FWD(float, false);
  }
#undef CYFA_LP_FWD
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
