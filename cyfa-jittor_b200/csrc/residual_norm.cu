// Residual add of a block's branch with the norms on both sides of it:
//   z  = y                      or  y / rms(y) * post      (post-norm)
//   x' = x + scale sigmoid(gate) z   (rounded to x's type; absent factors are 1)
//   h  = x' / rms(x') * weight       (the next branch's input)
// with rms(a) = sqrt(mean(a^2) + eps), and its backward pass: with dx', dh given,
//   dt    = dx' + (dh weight - x^ mean(dh weight x^)) / rms(x'),  x^ = x' / rms(x')
//   dx    = dt,   dz = dt scale sigmoid(gate)
//   dgate = dt scale z sigmoid(gate) (1 - sigmoid(gate)),  dscale = sum dt sigmoid(gate) z
//   dy    = dz    or  (dz post - y^ mean(dz post y^)) / rms(y)
//   dweight = sum dh x^,   dpost = sum dz y^   (over the rows)
// The arithmetic is fp32, but for the branch of bf16 rows ahead of x', which is carried in
// pairs of fp32 numbers with its row sums in 64 bits (below).  Each thread owns E columns
// of a row (kept in registers between the reductions and the stores), so every tensor is
// read and written once; column sums go through per-CTA partial rows added in a fixed order.
// Bound by memory for 16-byte rows: 16384 x 1024 bf16, the plain sum, 22 us forward
// (134 MB at 6.1 TB/s) and 35 us backward (the same bytes at 3.8: a row's two reductions
// stand between its loads and its stores); the sums of the partial rows take 3 us.
// Rows at any alignment are bound by the issue of one access an entry: 4099 x 1531 f32
// with both norms, gate and scale 34 us forward and 55 backward (125 and 201 MB).  bf16
// rows with a gate are bound by the arithmetic of the pairs (below): 16384 x 1024 with
// post-norm and gate 93 us forward (168 MB); 90 backward (268 MB), which has no pairs.
#include <algorithm>

#include "cyfa_common.cuh"

namespace cyfa {

constexpr int kRnMaxWidth = 8192;  // 1024 threads
constexpr int kRnFewRows = 4096;  // bf16 rows that are taken 8 columns a thread

struct ResNormParams {
  const void *x, *y, *gate;          // [rows, D], strides below; y and gate may be null
  long long sx, sy, sgate;           // row strides in elements
  const float *weight, *post;        // [D]; post may be null
  const float* scale_v;              // [D] or null
  float scale;                       // when scale_v is null
  float eps;
  long long rows;
  int D;
  void *xn, *h;                      // [rows, D] contiguous; xn null when y is null
  float *rstd_x, *rstd_y;            // [rows]; rstd_y null without post
  // backward
  const void *dxn, *dh;              // [rows, D] contiguous, may be null
  void *dx, *dy, *dgate;             // [rows, D] contiguous, may be null
  float* part;                       // [CTAs][3][D] column sums: dweight, dpost, dscale
  int stages;                        // shared-memory slots of a streamed row: 2, or 1 (no copy ahead)
};

// A thread's 8 columns threadIdx.x + j TX of a row, for single elements (TX threads a
// row, known to the compiler: the columns are then immediate offsets).
template <typename T, int TX>
struct RnRow {
  static constexpr int E = 8;
  int left;  // columns of the row from the thread's first on
  __device__ __forceinline__ explicit RnRow(int D) : left(D - int(threadIdx.x)) {}
  // p: the row, or null for zeros; n: left, or 0 for a row past the end
  __device__ __forceinline__ void load(const T* p, int n, float (&f)[E]) const {
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = 0.f;
    if (p) {
      p += threadIdx.x;
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (j * TX < n) f[j] = float(p[j * TX]);
    }
  }
  __device__ __forceinline__ void param(const float* p, float (&f)[E]) const {
    p += threadIdx.x;
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = j * TX < left ? __ldg(p + j * TX) : 0.f;
  }
  __device__ __forceinline__ void store(T* p, int n, const float (&f)[E]) const {
    p += threadIdx.x;
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j * TX < n) p[j * TX] = T(f[j]);
  }
};
template <typename T>
__device__ __forceinline__ const T* rn_at(const void* base, long long off) {
  return base ? static_cast<const T*>(base) + off : nullptr;
}

// Sum over the threads of one row (threadIdx.x), the same in all of them and in
// the same order.  red: one float per warp of the CTA.
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = int(blockDim.x) >> 5;
  if (warps == 1) return v;
  red += threadIdx.y * warps;
  __syncthreads();  // the last sum has been read
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < warps; ++w) s += red[w];
  return s;
}

// Branch arithmetic.  A bf16 stream is normalised after it is rounded, so every error
// of x' before that rounding moves some entries to the neighbouring bf16 value, 2^-8
// off: with plain fp32 arithmetic one entry in 2^16, which is what then limits
// dweight's distance from the exact sum (1e-5 relative on average, 2e-4 for a few rows
// where one entry moves; exact x': 1e-7).  For bf16 rows the branch is
// therefore carried in pairs of fp32 numbers (value + error: 2^-29 with a gate, 2^-40
// without), and x' is the exact sum's rounding but for one entry in 10^7 (16.7 M
// entries: 0 or 1 off, against 220 to 560 of the plain formula).  fp32 rows use single
// numbers.
struct Pair {
  float h, l;
};
__device__ __forceinline__ Pair pair_mul(Pair a, float b) {
  const float h = a.h * b;
  return Pair{h, fmaf(a.l, b, fmaf(a.h, b, -h))};
}
__device__ __forceinline__ Pair pair_mul(Pair a, Pair b) {
  const float h = a.h * b.h;
  return Pair{h, fmaf(a.h, b.l, fmaf(a.l, b.h, fmaf(a.h, b.h, -h)))};
}
// x + a, rounded once; an infinite sum has no error to add (its parts are NaN)
__device__ __forceinline__ float pair_add(float x, Pair a) {
  const float s = x + a.h, b = s - x;
  const float r = s + (((x - (s - b)) + (a.h - b)) + a.l);
  return fabsf(s) == INFINITY ? s : r;
}
// 1 / (1 + e^-z).  e^-z = 2^k e^r with r = -z - k ln 2 in [-0.35, 0.35] (ln 2 split after
// Cody and Waite, k ln2_hi exact) and e^r from its Taylor series, the terms up to
// r^2 / 2 in pairs, the rest (below 2^-7) in fp32.
__device__ __forceinline__ Pair pair_sigmoid(float z) {
  const float a = fminf(fmaxf(-z, -87.f), 87.f);  // (NaN: any)
  const float k = rintf(a * 1.44269504f);
  // ln 2 = 45426 / 65536 + 1.4286068e-6
  const float r0 = fmaf(-k, 0.693145751953125f, a);
  const float p = k * 1.42860682e-6f;
  const float rh = r0 - p, rl = (r0 - rh) - p;
  const float qh = rh * rh, ql = fmaf(rh, rh, -qh) + 2.f * rh * rl;
  // r^3 (1/6 + r/24 + r^2/120 + ... + r^7 / 10!)
  float c = 2.7557319e-7f;
  c = fmaf(c, rh, 2.7557319e-6f);
  c = fmaf(c, rh, 2.4801587e-5f);
  c = fmaf(c, rh, 1.9841270e-4f);
  c = fmaf(c, rh, 1.3888889e-3f);
  c = fmaf(c, rh, 8.3333333e-3f);
  c = fmaf(c, rh, 4.1666667e-2f);
  c = fmaf(c, rh, 1.6666667e-1f);
  c *= qh * rh;
  // e^r = 1 + r + r^2 / 2 + c as a pair
  const float s1 = 1.f + rh, t1 = rh - (s1 - 1.f);
  const float s2 = s1 + 0.5f * qh, t2 = 0.5f * qh - (s2 - s1);
  const float s3 = s2 + c, t3 = c - (s3 - s2);
  const float low = ((t1 + t2) + t3) + (rl + 0.5f * ql);
  const float two_k = __int_as_float((int(k) + 127) << 23);
  const float eh = s3 * two_k, el = low * two_k;
  // 1 / (1 + e): a quotient and its remainder
  const float d = 1.f + eh;
  const float dl = (eh > 1.f ? (1.f - (d - eh)) : (eh - (d - 1.f))) + el;
  const float g = __frcp_rn(d);
  const float rem = fmaf(-dl, g, fmaf(-d, g, 1.f));
  return z >= -87.f ? Pair{g, g * rem} : Pair{z != z ? z : 0.f, 0.f};
}
__device__ __forceinline__ float rn_gate(float z) { return 1.f / (1.f + expf(-z)); }
// sigmoid(z) and 1 - sigmoid(z) for the gradients.  fp32 rows: both to a few ulp for any
// z (1 - q cancels, and ex2.approx of a rounded z log2 e is 2^-18 off at |z| = 80): 96 us
// against 93 for 16384 x 1024 with a gate, backward, and 106 with a quotient in place of
// rcp.approx, which is 2^-23 off at most.  bf16 rows: the approximate instructions, 2^-20
// off where |z| < 16, far inside the gradients' rounding to 2^-8.
template <typename T>
__device__ __forceinline__ void rn_gate_pair(float z, float& q, float& rest) {
  if (sizeof(T) == 4) {
    const float e = expf(-fabsf(z));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    const float er = e * r;
    q = z >= 0.f ? r : er;
    rest = z >= 0.f ? er : r;
  } else {
    q = sigmoid_mufu(z);
    rest = 1.f - q;
  }
}

// Sum of squares of bf16 values (exact products), as a pair.
__device__ __forceinline__ void pair_square(float y, float& s, float& c) {
  const float q = y * y, t = s + q, b = t - s;
  c += (s - (t - b)) + (q - b);
  s = t;
}
// row_sum of pairs, in 64 bits
__device__ __forceinline__ double row_sum_pair(float s, float c, double* red) {
  double v = s == INFINITY ? double(s) : double(s) + double(c);
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = int(blockDim.x) >> 5;
  if (warps == 1) return v;
  red += threadIdx.y * warps;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < warps; ++w) v += red[w];
  return v;
}
__device__ __forceinline__ Pair pair_of(double v) {
  const float h = float(v);
  return Pair{h, float(v - double(h))};
}

template <typename T>
__device__ __forceinline__ float rn_round(float v) {
  return float(T(v));
}

// ------------------------------------------------ streamed rows
// Persistent CTAs of blockDim (threads of a row, rows at a time).  Each thread copies
// its E columns of the next row into its own shared-memory slots (cp.async, no
// barrier: nobody else reads them) while it works on the current one, so that the
// loads never wait for a row's sums and cost no registers.
template <typename T, int E>
struct RnStream {
  static constexpr int VEC = 16 / sizeof(T), J = E / VEC;
  uint32_t slot;     // shared address of the thread's first chunk
  int threads, tensors;
  int c0, cs;        // columns c0 + j cs ..
  uint32_t mask;     // chunks inside the row
  __device__ __forceinline__ RnStream(void* smem, int tensors_, int D)
      : threads(int(blockDim.x * blockDim.y)), tensors(tensors_), c0(int(threadIdx.x) * VEC),
        cs(int(blockDim.x) * VEC), mask(0) {
    slot = smem_u32(smem) + (threadIdx.y * blockDim.x + threadIdx.x) * 16;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (c0 + j * cs < D) mask |= 1u << j;
  }
  __device__ __forceinline__ uint32_t at(int stage, int tensor, int j) const {
    return slot + ((stage * tensors + tensor) * J + j) * threads * 16;
  }
  // row: at this thread's first column, or null for zeros
  __device__ __forceinline__ void copy(int stage, int tensor, const T* row, uint32_t m) const {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const bool ok = row && ((m >> j) & 1);
      cp_async16(at(stage, tensor, j), ok ? row + j * cs : row, ok);
    }
  }
  __device__ __forceinline__ void get(int stage, int tensor, int j, float* f) const {
    LpVec<T>::unpack(ld_shared_v4(at(stage, tensor, j)), f);
  }
  __device__ __forceinline__ void param(const float* p, int j, float* f) const {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 v = (mask >> j) & 1 ? __ldg(reinterpret_cast<const float4*>(p + c0 + j * cs + i))
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
      f[i] = v.x;
      f[i + 1] = v.y;
      f[i + 2] = v.z;
      f[i + 3] = v.w;
    }
  }
  static __device__ __forceinline__ void store(T* p, const uint4& u) {
    *reinterpret_cast<uint4*>(p) = u;
  }
};

// PLAIN: y alone, no post-norm, gate or scale.
template <typename T, int E, bool PLAIN>
__global__ void __launch_bounds__(256) residual_norm_fwd_stream_kernel(ResNormParams p) {
  using S = RnStream<T, E>;
  constexpr int VEC = S::VEC, J = S::J;
  extern __shared__ __align__(16) uint8_t rn_smem[];
  __shared__ float red[32];
  __shared__ double red64[32];
  pdl_wait();
  pdl_trigger();
  const int D = p.D;
  const S st(rn_smem, PLAIN ? 2 : 1 + (p.y != nullptr) + (p.gate != nullptr), D);
  const long long step = (long long)gridDim.x * blockDim.y;
  auto fetch = [&](long long row, int stage) {
    const uint32_t m = row < p.rows ? st.mask : 0;
    st.copy(stage, 0, rn_at<T>(p.x, row * p.sx + st.c0), m);
    if (PLAIN || p.y) st.copy(stage, 1, rn_at<T>(p.y, row * p.sy + st.c0), m);
    if (!PLAIN && p.gate) st.copy(stage, 2, rn_at<T>(p.gate, row * p.sgate + st.c0), m);
    cp_async_commit();
  };
  long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const int flip = p.stages - 1;
  if (flip) fetch(row, 0);
  for (int s = 0; row - threadIdx.y < p.rows; row += step, s ^= flip) {
    fetch(flip ? row + step : row, s ^ flip);
    if (flip) cp_async_wait<1>(); else cp_async_wait<0>();
    const uint32_t m = row < p.rows ? st.mask : 0;
    const bool first = row < p.rows && threadIdx.x == 0;
    T* xn = static_cast<T*>(p.xn) + row * D + st.c0;
    T* h = static_cast<T*>(p.h) + row * D + st.c0;
    constexpr bool PAIRS = sizeof(T) == 2;
    float rsy = 1.f;
    Pair rsp{1.f, 0.f};
    if (!PLAIN && p.post) {
      float ss = 0.f, sc = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float y[VEC];
        st.get(s, 1, j, y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (PAIRS) pair_square(y[i], ss, sc); else ss = fmaf(y[i], y[i], ss);
        }
      }
      if (PAIRS) {
        rsp = pair_of(1.0 / sqrt(row_sum_pair(ss, sc, red64) / D + double(p.eps)));
        rsy = rsp.h;
      } else {
        rsy = __frsqrt_rn(row_sum(ss, red) / D + p.eps);
      }
      if (first && p.rstd_y) p.rstd_y[row] = rsy;
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float t[VEC];
      st.get(s, 0, j, t);
      if (PLAIN || p.y) {
        float z[VEC];
        st.get(s, 1, j, z);
        if (PLAIN) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) t[i] += z[i];
        } else {
          float w[VEC], g[VEC], sc[VEC];
          if (p.post) st.param(p.post, j, w);
          if (p.gate) st.get(s, 2, j, g);
          if (p.scale_v) st.param(p.scale_v, j, sc);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float scale = p.scale_v ? sc[i] : p.scale;
            if (PAIRS) {
              Pair u{z[i], 0.f};
              if (p.post) u = pair_mul(pair_mul(rsp, z[i]), w[i]);
              if (p.gate) u = pair_mul(u, pair_sigmoid(g[i]));
              t[i] = pair_add(t[i], pair_mul(u, scale));
            } else {
              float u = z[i];
              if (p.post) u = u * rsy * w[i];
              if (p.gate) u *= rn_gate(g[i]);
              t[i] = fmaf(scale, u, t[i]);
            }
          }
        }
        // the norm reads the stream as it is kept, in x's type
        const uint4 u = LpVec<T>::pack(t);
        LpVec<T>::unpack(u, t);
        st_shared_v4(st.at(s, 0, j), u.x, u.y, u.z, u.w);
        if ((m >> j) & 1) S::store(xn + j * st.cs, u);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = fmaf(t[i], t[i], ss);
    }
    const float rs = __frsqrt_rn(row_sum(ss, red) / D + p.eps);
    if (first && p.rstd_x) p.rstd_x[row] = rs;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float t[VEC], w[VEC];
      st.get(s, 0, j, t);
      st.param(p.weight, j, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = t[i] * rs * w[i];
      if ((m >> j) & 1) S::store(h + j * st.cs, LpVec<T>::pack(t));
    }
  }
  cp_async_wait<0>();
}

// The column sums of a CTA's threads (dweight and, with FULL, dpost and dscale): its
// row slots side by side in shared memory [rows][D], then added in order, as one
// partial row.
template <int SETS, typename Put>
__device__ __forceinline__ void rn_partial(float* out, float* buf, int D, Put put) {
  const int tid = int(threadIdx.y * blockDim.x + threadIdx.x), n = int(blockDim.x * blockDim.y);
#pragma unroll
  for (int k = 0; k < SETS; ++k) {
    __syncthreads();
    put(k, buf + threadIdx.y * D);
    __syncthreads();
    for (int c = tid; c < D; c += n) {
      float v = buf[c];
      for (int y = 1; y < int(blockDim.y); ++y) v += buf[y * D + c];
      out[k * D + c] = v;
    }
  }
}

// p.x is the new stream x'.  FULL: with y's side; otherwise dx alone (the plain sum's
// dy equals it).
template <typename T, int E, bool FULL>
__global__ void __launch_bounds__(256) residual_norm_bwd_stream_kernel(ResNormParams p) {
  using S = RnStream<T, E>;
  constexpr int VEC = S::VEC, J = S::J;
  extern __shared__ __align__(16) uint8_t rn_smem[];
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const int D = p.D;
  const S st(rn_smem, FULL ? 4 + (p.gate != nullptr) : 3, D);
  const float inv = 1.f / D;
  const long long step = (long long)gridDim.x * blockDim.y;
  auto fetch = [&](long long row, int stage) {
    const uint32_t m = row < p.rows ? st.mask : 0;
    st.copy(stage, 0, rn_at<T>(p.x, row * p.sx + st.c0), m);
    st.copy(stage, 1, rn_at<T>(p.dh, row * D + st.c0), m);
    st.copy(stage, 2, rn_at<T>(p.dxn, row * D + st.c0), m);
    if (FULL) {
      st.copy(stage, 3, rn_at<T>(p.y, row * p.sy + st.c0), m);
      if (p.gate) st.copy(stage, 4, rn_at<T>(p.gate, row * p.sgate + st.c0), m);
    }
    cp_async_commit();
  };
  float acc[FULL ? 3 : 1][E];  // dweight, dpost, dscale
#pragma unroll
  for (int k = 0; k < (FULL ? 3 : 1); ++k)
#pragma unroll
    for (int i = 0; i < E; ++i) acc[k][i] = 0.f;
  long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const int flip = p.stages - 1;
  if (flip) fetch(row, 0);
  for (int s = 0; row - threadIdx.y < p.rows; row += step, s ^= flip) {
    fetch(flip ? row + step : row, s ^ flip);
    const bool in = row < p.rows;
    const uint32_t m = in ? st.mask : 0;
    const float rs = in ? p.rstd_x[row] : 0.f;
    const float rsy = FULL && p.post && in ? p.rstd_y[row] : 1.f;
    if (flip) cp_async_wait<1>(); else cp_async_wait<0>();
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float t[VEC], g[VEC], w[VEC];
      st.get(s, 0, j, t);
      st.get(s, 1, j, g);
      st.param(p.weight, j, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float gt = g[i] * t[i];  // rs, the same for the row, comes in once below
        acc[0][j * VEC + i] = fmaf(gt, rs, acc[0][j * VEC + i]);
        dot = fmaf(gt, w[i], dot);
      }
    }
    // dt = dxn + rs g w - t rs^2 dot
    dot = row_sum(dot * rs, red) * inv * rs * rs;
    float dz[FULL ? E : 1], doty = 0.f;
    T* dx = static_cast<T*>(p.dx) + row * D + st.c0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float t[VEC], g[VEC], dt[VEC], w[VEC];
      st.get(s, 0, j, t);
      st.get(s, 1, j, g);
      st.get(s, 2, j, dt);
      st.param(p.weight, j, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) dt[i] = fmaf(g[i] * w[i], rs, fmaf(-dot, t[i], dt[i]));
      if (p.dx && ((m >> j) & 1)) S::store(dx + j * st.cs, LpVec<T>::pack(dt));
      if constexpr (FULL) {
        float y[VEC], f[VEC], sc[VEC], sg[VEC];
        st.get(s, 3, j, y);
        if (p.scale_v) {
          st.param(p.scale_v, j, sc);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) sc[i] = p.scale;
        }
        if (p.post) {
          st.param(p.post, j, f);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) f[i] = 1.f;
        }
        if (p.gate) {
          st.get(s, 4, j, sg);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float q, rest;
            rn_gate_pair<T>(sg[i], q, rest);
            const float d = dt[i] * q;
            sg[i] = d * sc[i] * (y[i] * rsy * f[i]) * rest;
            dt[i] = d;
          }
          if (p.dgate && ((m >> j) & 1))
            S::store(static_cast<T*>(p.dgate) + row * D + st.c0 + j * st.cs, LpVec<T>::pack(sg));
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float yh = y[i] * rsy, d = dt[i] * sc[i], e = d * f[i];
          acc[2][j * VEC + i] = fmaf(dt[i], yh * f[i], acc[2][j * VEC + i]);
          acc[1][j * VEC + i] = fmaf(d, yh, acc[1][j * VEC + i]);
          doty = fmaf(e, yh, doty);
          dz[j * VEC + i] = e;
        }
      }
    }
    if constexpr (FULL) {
      if (p.post) doty = row_sum(doty, red) * inv;
      T* dy = static_cast<T*>(p.dy) + row * D + st.c0;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float y[VEC];
        if (p.post) {
          st.get(s, 3, j, y);
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[i] = rsy * fmaf(-y[i] * rsy, doty, dz[j * VEC + i]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[i] = dz[j * VEC + i];
        }
        if (p.dy && ((m >> j) & 1)) S::store(dy + j * st.cs, LpVec<T>::pack(y));
      }
    }
  }
  cp_async_wait<0>();
  rn_partial<FULL ? 3 : 1>(
      p.part + (long long)blockIdx.x * 3 * D, reinterpret_cast<float*>(rn_smem), D,
      [&](int k, float* row_buf) {
#pragma unroll
        for (int j = 0; j < J; ++j)
          if ((st.mask >> j) & 1) {
            float* q = row_buf + st.c0 + j * st.cs;
#pragma unroll
            for (int i = 0; i < VEC; ++i) q[i] = acc[k][j * VEC + i];
          }
      });
}

// ------------------------------------------------ rows at any alignment
// Persistent CTAs as above, a thread's 8 columns TX apart, all of a row's loads ahead
// of its sums.  What bounds these is the issue of one access an element; 4-byte
// asynchronous copies into shared memory in their place took 55 and 126 us (forward
// and backward, 4099 x 1531 fp32 with both norms, gate and scale).
template <typename T, int TX>
__global__ void __launch_bounds__(TX > 256 ? TX : 256, TX > 256 ? 1 : 4)
    residual_norm_fwd_kernel(ResNormParams p) {
  using R = RnRow<T, TX>;
  constexpr int E = R::E;
  pdl_wait();
  pdl_trigger();
  __shared__ float red[32];
  __shared__ double red64[32];
  const int D = p.D;
  const R r(D);
  for (long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y; row - threadIdx.y < p.rows;
       row += (long long)gridDim.x * blockDim.y) {
    // rows past the end take part in the barriers only
    const int m = row < p.rows ? r.left : 0;
    const bool first = row < p.rows && threadIdx.x == 0;
    float t[E], z[E], g[E];
    r.load(rn_at<T>(p.x, row * p.sx), m, t);
    r.load(rn_at<T>(p.y, row * p.sy), m, z);
    r.load(rn_at<T>(p.gate, row * p.sgate), m, g);
    if (p.y) {
      constexpr bool PAIRS = sizeof(T) == 2;
      float w[E], sv[E], rsy = 1.f;
      Pair rsp{1.f, 0.f};
      if (p.post) {
        float ss = 0.f, sc = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if (PAIRS) pair_square(z[i], ss, sc); else ss = fmaf(z[i], z[i], ss);
        }
        if (PAIRS) {
          rsp = pair_of(1.0 / sqrt(row_sum_pair(ss, sc, red64) / D + double(p.eps)));
          rsy = rsp.h;
        } else {
          rsy = __frsqrt_rn(row_sum(ss, red) / D + p.eps);
        }
        r.param(p.post, w);
        if (first && p.rstd_y) p.rstd_y[row] = rsy;
      }
      if (p.scale_v) r.param(p.scale_v, sv);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float scale = p.scale_v ? sv[i] : p.scale;
        if (PAIRS) {
          Pair u{z[i], 0.f};
          if (p.post) u = pair_mul(pair_mul(rsp, z[i]), w[i]);
          if (p.gate) u = pair_mul(u, pair_sigmoid(g[i]));
          t[i] = pair_add(t[i], pair_mul(u, scale));
        } else {
          float u = z[i];
          if (p.post) u = u * rsy * w[i];
          if (p.gate) u *= rn_gate(g[i]);
          t[i] = fmaf(scale, u, t[i]);
        }
        t[i] = rn_round<T>(t[i]);  // the norm reads the stream as it is kept, in x's type
      }
      r.store(static_cast<T*>(p.xn) + row * D, m, t);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) ss = fmaf(t[i], t[i], ss);
    const float rs = __frsqrt_rn(row_sum(ss, red) / D + p.eps);
    if (first && p.rstd_x) p.rstd_x[row] = rs;
    r.param(p.weight, g);
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] = t[i] * rs * g[i];
    r.store(static_cast<T*>(p.h) + row * D, m, t);
  }
}

// p.x is the new stream x'.
template <typename T, int TX, bool FULL>
__global__ void __launch_bounds__(TX > 256 ? TX : 256, TX > 256 ? 1 : (FULL ? 2 : 3))
    residual_norm_bwd_kernel(ResNormParams p) {
  using R = RnRow<T, TX>;
  constexpr int E = R::E;
  extern __shared__ __align__(16) uint8_t rn_smem[];
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const int D = p.D;
  const R r(D);
  float acc[FULL ? 3 : 1][E];  // dweight, dpost, dscale
#pragma unroll
  for (int k = 0; k < (FULL ? 3 : 1); ++k)
#pragma unroll
    for (int i = 0; i < E; ++i) acc[k][i] = 0.f;
  const float inv = 1.f / D;
  for (long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y; row - threadIdx.y < p.rows;
       row += (long long)gridDim.x * blockDim.y) {
    const bool in = row < p.rows;
    const int m = in ? r.left : 0;
    float t[E], g[E], dt[E], y[E], sg[E], w[E];
    r.load(rn_at<T>(p.x, row * p.sx), m, t);
    r.load(rn_at<T>(p.dh, row * D), m, g);
    r.load(rn_at<T>(p.dxn, row * D), m, dt);
    if (FULL) {
      r.load(rn_at<T>(p.y, row * p.sy), m, y);
      r.load(rn_at<T>(p.gate, row * p.sgate), m, sg);
    }
    const float rs = in ? p.rstd_x[row] : 0.f;
    const float rsy = FULL && p.post && in ? p.rstd_y[row] : 1.f;
    r.param(p.weight, w);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      t[i] *= rs;
      acc[0][i] = fmaf(g[i], t[i], acc[0][i]);
      g[i] *= w[i];
      dot = fmaf(g[i], t[i], dot);
    }
    dot = row_sum(dot, red) * inv;
#pragma unroll
    for (int i = 0; i < E; ++i) dt[i] = fmaf(rs, fmaf(-t[i], dot, g[i]), dt[i]);
    if (p.dx) r.store(static_cast<T*>(p.dx) + row * D, m, dt);
    if constexpr (FULL) {
      // t: scale, w: post weight, g: gate
      if (p.scale_v) {
        r.param(p.scale_v, t);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) t[i] = p.scale;
      }
      if (p.post) {
        r.param(p.post, w);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = 1.f;
      }
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] *= rsy;
      if (p.gate) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float q, rest;
          rn_gate_pair<T>(sg[i], q, rest);
          dt[i] *= q;
          sg[i] = dt[i] * t[i] * (y[i] * w[i]) * rest;
        }
        if (p.dgate) r.store(static_cast<T*>(p.dgate) + row * D, m, sg);
      }
      float doty = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        acc[2][i] = fmaf(dt[i], y[i] * w[i], acc[2][i]);
        dt[i] *= t[i];
        acc[1][i] = fmaf(dt[i], y[i], acc[1][i]);
        dt[i] *= w[i];
        doty = fmaf(dt[i], y[i], doty);
      }
      if (p.post) {
        doty = row_sum(doty, red) * inv;
#pragma unroll
        for (int i = 0; i < E; ++i) dt[i] = rsy * fmaf(-y[i], doty, dt[i]);
      }
      if (p.dy) r.store(static_cast<T*>(p.dy) + row * D, m, dt);
    }
  }
  rn_partial<FULL ? 3 : 1>(p.part + (long long)blockIdx.x * 3 * D, reinterpret_cast<float*>(rn_smem), D,
                           [&](int k, float* row_buf) {
#pragma unroll
                             for (int j = 0; j < E; ++j)
                               if (j * TX < r.left) row_buf[threadIdx.x + j * TX] = acc[k][j];
                           });
}

// Column sums of the partial rows, in a fixed order: CTA (32 columns, set),
// 32 row strides, then a fixed tree.
__global__ void __launch_bounds__(1024)
    residual_norm_sum_kernel(const float* part, int n, int D, float* dweight, float* dpost,
                             float* dscale) {
  pdl_wait();
  pdl_trigger();
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x, set = blockIdx.y;
  float* out = set == 0 ? dweight : (set == 1 ? dpost : dscale);
  if (!out) return;
  float acc = 0.f;
  if (c < D)
    for (int r = threadIdx.y; r < n; r += 32) acc += part[((size_t)r * 3 + set) * D + c];
  s[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  float v = s[threadIdx.x][threadIdx.y];  // row strides of column blockIdx.x * 32 + threadIdx.y
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int cc = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && cc < D) out[cc] = v;
}

// Columns of a thread: 8, which leaves the most room for rows in flight, unless bf16 rows
// are many enough that 32, a row of 1024 to a warp, saves more in barriers, or a row
// would not fit 256 threads; with y's side 16 for the three accumulators a column.
// Backward times in us: bf16 rows of 1024, plain, 4096 of them 20 with 8 and 23 with 32,
// 16384 of them 46 and 42, with post-norm and gate 114 and 97; 4096 x 4096 with both 113
// with 16, 120 with 32; f32 8192 x 2048 with both 114 with 8, 139 with 16, 4096 x 4096
// plain 62 with 16, 66 with 32.
static int rn_elems(int D, int es, long long rows, bool vector, bool full) {
  if (!vector || D <= 256) return 8;
  if (es == 4) return D <= 2048 ? 8 : (D <= 4096 ? 16 : 32);
  if (D <= 2048 && rows <= kRnFewRows) return 8;
  return full && D > 1024 && D <= 4096 ? 16 : 32;
}
// threads of a row with E columns each, and rows of a CTA
static dim3 rn_block(int D, int E, bool vector, long long rows) {
  int tx = ((D + E - 1) / E + 31) / 32 * 32;
  if (!vector) {  // the spacings that are built
    int t = 32;
    while (t < tx) t = t == 256 ? 1024 : 2 * t;
    tx = t;
  }
  int ty = 1;
  while (ty < 8 && tx * ty * 2 <= 256 && rows > ty) ty *= 2;
  return dim3(unsigned(tx), unsigned(ty));
}
// shared memory of one slot of a row's tensors; two slots where they fit (they do not
// for four or five fp32 tensors of more than 5600 columns)
static size_t rn_slot_bytes(dim3 block, int elems, int es, int tensors) {
  return size_t(tensors) * elems * es * block.x * block.y;
}
constexpr int kRnMaxSmem = 226 << 10;
static int rn_stages(size_t slot) { return 2 * slot <= kRnMaxSmem ? 2 : 1; }
// CTAs an SM holds at a time (shared memory and registers)
static int rn_per_sm(dim3 block, bool vector, size_t smem) {
  const int threads = int(block.x * block.y);
  if (!vector) return std::max(1, 1024 / threads);
  return int(std::max<size_t>(1, std::min<size_t>(std::min<size_t>(4, 768 / threads),
                                                  (220 << 10) / (smem + 1024))));
}
struct RnBwdShape {
  int elems, stages;
  dim3 block;
  size_t smem;
  unsigned grid;
  RnBwdShape(int D, int es, long long rows, bool full, bool gate, bool vector) {
    elems = rn_elems(D, es, rows, vector, full);
    block = rn_block(D, elems, vector, rows);
    const size_t slot = rn_slot_bytes(block, elems, es, full ? 4 + gate : 3);
    stages = rn_stages(slot);
    smem = vector ? stages * slot : block.y * D * sizeof(float);
    grid = unsigned(std::min<long long>((rows + block.y - 1) / block.y,
                                        148ll * rn_per_sm(block, vector, smem)));
  }
};

// Whether every row and parameter allows 16-byte accesses.
static bool rn_vector(int D, int es, std::initializer_list<const void*> ptrs,
                      std::initializer_list<const float*> params,
                      std::initializer_list<long long> strides) {
  bool ok = D * es % 16 == 0;
  for (const void* q : ptrs) ok = ok && aligned(q, 16);
  for (const float* q : params) ok = ok && aligned(q, 16);
  for (long long st : strides) ok = ok && st * es % 16 == 0;
  return ok;
}

static int rn_checks(int dtype, long long rows, int D) {
  CYFA_REQUIRE(rows > 0 && rows < (1ll << 31) && D > 0 && D <= kRnMaxWidth, kBadShape);
  CYFA_REQUIRE(dtype == 0 || dtype == 1, kBadDtype);
  return kOk;
}

}  // namespace cyfa

extern "C" {

int cyfa_residual_norm_fwd(const cyfa_residual_norm_args* a, void* xn, void* h, float* rstd_x,
                           float* rstd_y, void* stream) {
  CYFA_REQUIRE(a && a->x && a->weight && h && (!a->y || xn) &&
                   (!a->post_weight || a->y) && (!a->gate || a->y),
               kNullPointer);
  const int rc = rn_checks(a->dtype, a->rows, a->D);
  if (rc) return rc;
  const int es = a->dtype == 1 ? 2 : 4;
  for (const void* q : {a->x, a->y, a->gate, (const void*)xn, (const void*)h})
    CYFA_REQUIRE(aligned(q, es), kMisaligned);
  ResNormParams p{};
  p.x = a->x;
  p.y = a->y;
  p.gate = a->gate;
  p.sx = a->x_stride;
  p.sy = a->y_stride;
  p.sgate = a->gate_stride;
  p.weight = a->weight;
  p.post = a->post_weight;
  p.scale_v = a->scale_vector;
  p.scale = a->scale;
  p.eps = a->eps;
  p.rows = a->rows;
  p.D = a->D;
  p.xn = xn;
  p.h = h;
  p.rstd_x = rstd_x;
  p.rstd_y = rstd_y;
  const bool vector = rn_vector(a->D, es, {a->x, a->y, a->gate, xn, h},
                                {a->weight, a->post_weight, a->scale_vector},
                                {a->x_stride, a->y ? a->y_stride : 0, a->gate ? a->gate_stride : 0});
  const int elems = rn_elems(a->D, es, a->rows, vector, false);
  const dim3 block = rn_block(a->D, elems, vector, a->rows);
  const long long ctas = (a->rows + block.y - 1) / block.y;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (vector) {
    const size_t slot = rn_slot_bytes(block, elems, es, 1 + (a->y != nullptr) + (a->gate != nullptr));
    p.stages = rn_stages(slot);
    const size_t smem = p.stages * slot;
    const unsigned grid = unsigned(std::min<long long>(ctas, 148ll * rn_per_sm(block, vector, smem)));
    const bool plain = a->y && !a->post_weight && !a->gate && !a->scale_vector && a->scale == 1.f;
#define CYFA_RN_L(T, E, PLAIN)                                                                       \
  do {                                                                                               \
    set_smem(residual_norm_fwd_stream_kernel<T, E, PLAIN>, kRnMaxSmem);                              \
    CYFA_LAUNCH("residual_norm_fwd", s,                                                              \
                (launch_k(residual_norm_fwd_stream_kernel<T, E, PLAIN>, grid, block, smem, s, p)));  \
  } while (0)
#define CYFA_RN(T, E) \
  do { if (plain) CYFA_RN_L(T, E, true); else CYFA_RN_L(T, E, false); } while (0)
    if (a->dtype == 1) {
      if (elems == 8) CYFA_RN(__nv_bfloat16, 8); else CYFA_RN(__nv_bfloat16, 32);
    } else {
      if (elems == 8) CYFA_RN(float, 8);
      else if (elems == 16) CYFA_RN(float, 16);
      else CYFA_RN(float, 32);
    }
#undef CYFA_RN
#undef CYFA_RN_L
    return launch_status();
  }
  const unsigned grid = unsigned(std::min<long long>(ctas, 148ll * rn_per_sm(block, vector, 0)));
#define CYFA_RN_L(T, TX)               \
  CYFA_LAUNCH("residual_norm_fwd", s, \
              (launch_k(residual_norm_fwd_kernel<T, TX>, grid, block, 0, s, p)))
#define CYFA_RN(T)                              \
  do {                                          \
    if (block.x == 32) CYFA_RN_L(T, 32);        \
    else if (block.x == 64) CYFA_RN_L(T, 64);   \
    else if (block.x == 128) CYFA_RN_L(T, 128); \
    else if (block.x == 256) CYFA_RN_L(T, 256); \
    else CYFA_RN_L(T, 1024);                    \
  } while (0)
  if (a->dtype == 1) CYFA_RN(__nv_bfloat16); else CYFA_RN(float);
#undef CYFA_RN
#undef CYFA_RN_L
  return launch_status();
}

size_t cyfa_residual_norm_bwd_work_bytes(long long rows, int D) {
  if (rows <= 0 || D <= 0 || D > kRnMaxWidth) return 0;
  size_t most = 0;
  for (int k = 0; k < 16; ++k) {
    const RnBwdShape sh(D, k & 1 ? 2 : 4, rows, k & 2, k & 4, k & 8);
    most = std::max(most, size_t(sh.grid));
  }
  return most * 3 * D * sizeof(float);
}

int cyfa_residual_norm_bwd(const cyfa_residual_norm_args* a, const float* rstd_x,
                           const float* rstd_y, const void* dxn, const void* dh, void* dx,
                           void* dy, void* dgate, float* dweight, float* dpost, float* dscale,
                           void* work, size_t work_bytes, void* stream) {
  CYFA_REQUIRE(a && a->x && a->weight && rstd_x && work && (!a->post_weight || (a->y && rstd_y)) &&
                   (!a->gate || a->y) && (a->y || (!dy && !dgate && !dpost && !dscale)),
               kNullPointer);
  const int rc = rn_checks(a->dtype, a->rows, a->D);
  if (rc) return rc;
  const int es = a->dtype == 1 ? 2 : 4;
  for (const void* q : {a->x, a->y, a->gate, dxn, dh, (const void*)dx, (const void*)dy,
                        (const void*)dgate})
    CYFA_REQUIRE(aligned(q, es), kMisaligned);
  CYFA_REQUIRE(aligned(work, 16), kMisaligned);
  CYFA_REQUIRE(work_bytes >= cyfa_residual_norm_bwd_work_bytes(a->rows, a->D), kWorkspace);
  ResNormParams p{};
  p.x = a->x;
  p.y = a->y;
  p.gate = a->gate;
  p.sx = a->x_stride;
  p.sy = a->y_stride;
  p.sgate = a->gate_stride;
  p.weight = a->weight;
  p.post = a->post_weight;
  p.scale_v = a->scale_vector;
  p.scale = a->scale;
  p.eps = a->eps;
  p.rows = a->rows;
  p.D = a->D;
  p.rstd_x = const_cast<float*>(rstd_x);
  p.rstd_y = const_cast<float*>(rstd_y);
  p.dxn = dxn;
  p.dh = dh;
  p.dx = dx;
  p.dy = dy;
  p.dgate = dgate;
  p.part = static_cast<float*>(work);
  // without gate, scale and post-norm, dy equals dx: the plain sum's gradient
  const bool full = a->y && (dy || dgate || dpost || dscale);
  const bool vector = rn_vector(a->D, es, {a->x, a->y, a->gate, dxn, dh, dx, dy, dgate},
                                {a->weight, a->post_weight, a->scale_vector},
                                {a->x_stride, a->y ? a->y_stride : 0, a->gate ? a->gate_stride : 0});
  const RnBwdShape sh(a->D, es, a->rows, full, a->gate != nullptr, vector);
  p.stages = sh.stages;
  const dim3 block = sh.block;
  const unsigned grid = sh.grid;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define CYFA_RN_S(T, E, FULL)                                                                        \
  do {                                                                                               \
    set_smem(residual_norm_bwd_stream_kernel<T, E, FULL>, kRnMaxSmem);                               \
    CYFA_LAUNCH("residual_norm_bwd", s,                                                              \
                (launch_k(residual_norm_bwd_stream_kernel<T, E, FULL>, grid, block, sh.smem, s, p))); \
  } while (0)
#define CYFA_RN_L(T, TX, FULL)         \
  CYFA_LAUNCH("residual_norm_bwd", s, \
              (launch_k(residual_norm_bwd_kernel<T, TX, FULL>, grid, block, sh.smem, s, p)))
#define CYFA_RN(T, FULL)                                          \
  do {                                                            \
    if (vector && sh.elems == 8) CYFA_RN_S(T, 8, FULL);           \
    else if (vector && sh.elems == 16) CYFA_RN_S(T, 16, FULL);    \
    else if (vector) CYFA_RN_S(T, 32, FULL);                      \
    else if (block.x == 32) CYFA_RN_L(T, 32, FULL);               \
    else if (block.x == 64) CYFA_RN_L(T, 64, FULL);               \
    else if (block.x == 128) CYFA_RN_L(T, 128, FULL);             \
    else if (block.x == 256) CYFA_RN_L(T, 256, FULL);             \
    else CYFA_RN_L(T, 1024, FULL);                                \
  } while (0)
  if (a->dtype == 1) {
    if (full) CYFA_RN(__nv_bfloat16, true); else CYFA_RN(__nv_bfloat16, false);
  } else {
    if (full) CYFA_RN(float, true); else CYFA_RN(float, false);
  }
#undef CYFA_RN
#undef CYFA_RN_L
#undef CYFA_RN_S
  if (dweight || dpost || dscale)
    CYFA_LAUNCH("residual_norm_sum", s,
                (launch_k(residual_norm_sum_kernel, dim3(unsigned((a->D + 31) / 32), 3), dim3(32, 32),
                          0, s, p.part, int(grid), a->D, dweight, dpost, dscale)));
  return launch_status();
}

}  // extern "C"
