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
// All arithmetic is fp32.  Each thread owns 8 columns of a row (kept in
// registers between the reductions and the stores), so every tensor is read and
// written once; column sums go through per-CTA partial rows added in a fixed
// order.
#include <algorithm>

#include "cyfa_common.cuh"

namespace cyfa {

constexpr int kRnElems = 8;        // columns of a thread
constexpr int kRnMaxWidth = 8192;  // 1024 threads

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
};

// The 8 columns of thread t among n threads: VEC consecutive ones at
// (t + j n) VEC for j < 8 / VEC.
template <typename T, int VEC>
struct RnRow {
  static constexpr int J = kRnElems / VEC;
  static __device__ __forceinline__ int col(int j) {
    return (int(threadIdx.x) + j * int(blockDim.x)) * VEC;
  }
  static __device__ __forceinline__ void load(const void* base, long long off, int D, float* f) {
    const T* p = static_cast<const T*>(base) + off;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = col(j);
      if (c < D) {
        EmbVec<T, VEC>::load(p + c, f + j * VEC);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[j * VEC + i] = 0.f;
      }
    }
  }
  static __device__ __forceinline__ void load_f32(const float* p, int D, float* f) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = col(j);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[j * VEC + i] = c < D ? __ldg(p + c + i) : 0.f;
    }
  }
  static __device__ __forceinline__ void store(void* base, long long off, int D, const float* f) {
    T* p = static_cast<T*>(base) + off;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (col(j) < D) EmbVec<T, VEC>::store(p + col(j), f + j * VEC);
  }
};

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

__device__ __forceinline__ float rn_sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }

template <typename T>
__device__ __forceinline__ float rn_round(float v) {
  return float(T(v));
}

// blockDim (threads of a row, rows of a CTA)
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) residual_norm_fwd_kernel(ResNormParams p) {
  using R = RnRow<T, VEC>;
  pdl_wait();
  pdl_trigger();
  __shared__ float red[32];
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool in = row < p.rows;
  const int D = in ? p.D : 0;  // rows past the end take part in the barriers only
  float t[kRnElems];
  R::load(p.x, row * p.sx, D, t);
  if (p.y) {
    float z[kRnElems];
    R::load(p.y, row * p.sy, D, z);
    if (p.post) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) ss = fmaf(z[i], z[i], ss);
      const float rs = rsqrtf(row_sum(ss, red) / p.D + p.eps);
      float w[kRnElems];
      R::load_f32(p.post, D, w);
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) z[i] = z[i] * rs * w[i];
      if (in && threadIdx.x == 0 && p.rstd_y) p.rstd_y[row] = rs;
    }
    if (p.gate) {
      float g[kRnElems];
      R::load(p.gate, row * p.sgate, D, g);
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) z[i] *= rn_sigmoid(g[i]);
    }
    if (p.scale_v) {
      float s[kRnElems];
      R::load_f32(p.scale_v, D, s);
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) z[i] *= s[i];
    } else {
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) z[i] *= p.scale;
    }
    // the norm reads the stream as it is kept, in x's type
#pragma unroll
    for (int i = 0; i < kRnElems; ++i) t[i] = rn_round<T>(t[i] + z[i]);
    R::store(p.xn, row * p.D, D, t);
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kRnElems; ++i) ss = fmaf(t[i], t[i], ss);
  const float rs = rsqrtf(row_sum(ss, red) / p.D + p.eps);
  if (in && threadIdx.x == 0 && p.rstd_x) p.rstd_x[row] = rs;
  float w[kRnElems];
  R::load_f32(p.weight, D, w);
#pragma unroll
  for (int i = 0; i < kRnElems; ++i) t[i] = t[i] * rs * w[i];
  R::store(p.h, row * p.D, D, t);
}

// p.x is the new stream x' here (contiguous or strided by sx).  A CTA walks its
// rows with the column sums in registers.
template <typename T, int VEC, bool FULL>
__global__ void __launch_bounds__(1024) residual_norm_bwd_kernel(ResNormParams p) {
  using R = RnRow<T, VEC>;
  pdl_wait();
  pdl_trigger();
  __shared__ float red[32];
  float dw[kRnElems], dp[kRnElems], ds[kRnElems];
#pragma unroll
  for (int i = 0; i < kRnElems; ++i) dw[i] = dp[i] = ds[i] = 0.f;
  float w[kRnElems];
  R::load_f32(p.weight, p.D, w);
  const float inv = 1.f / p.D;
  for (long long r0 = (long long)blockIdx.x * blockDim.y; r0 < p.rows;
       r0 += (long long)gridDim.x * blockDim.y) {
    const long long row = r0 + threadIdx.y;
    const bool in = row < p.rows;
    const int D = in ? p.D : 0;
    float dt[kRnElems];
    if (p.dxn) {
      R::load(p.dxn, row * p.D, D, dt);
    } else {
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) dt[i] = 0.f;
    }
    if (p.dh) {
      float t[kRnElems], g[kRnElems];
      R::load(p.x, row * p.sx, D, t);
      R::load(p.dh, row * p.D, D, g);
      const float rs = in ? p.rstd_x[row] : 0.f;
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) {
        t[i] *= rs;
        dw[i] = fmaf(g[i], t[i], dw[i]);
        g[i] *= w[i];
        dot = fmaf(g[i], t[i], dot);
      }
      dot = row_sum(dot, red) * inv;
#pragma unroll
      for (int i = 0; i < kRnElems; ++i) dt[i] = fmaf(rs, g[i] - t[i] * dot, dt[i]);
    }
    if (p.dx) R::store(p.dx, row * p.D, D, dt);
    if (FULL) {
      float y[kRnElems], s[kRnElems], f[kRnElems];
      R::load(p.y, row * p.sy, D, y);
      const float rs = p.post && in ? p.rstd_y[row] : 1.f;
      if (p.scale_v) {
        R::load_f32(p.scale_v, D, s);
      } else {
#pragma unroll
        for (int i = 0; i < kRnElems; ++i) s[i] = p.scale;
      }
      // y becomes y^; f: the post weight
      if (p.post) {
        R::load_f32(p.post, D, f);
#pragma unroll
        for (int i = 0; i < kRnElems; ++i) y[i] *= rs;
      } else {
#pragma unroll
        for (int i = 0; i < kRnElems; ++i) f[i] = 1.f;
      }
      if (p.gate) {
        float g[kRnElems];
        R::load(p.gate, row * p.sgate, D, g);
#pragma unroll
        for (int i = 0; i < kRnElems; ++i) {
          const float sg = rn_sigmoid(g[i]);
          g[i] = dt[i] * s[i] * y[i] * f[i] * (sg * (1.f - sg));
          ds[i] = fmaf(dt[i] * sg, y[i] * f[i], ds[i]);
          dt[i] *= s[i] * sg;  // dz from here on
        }
        if (p.dgate) R::store(p.dgate, row * p.D, D, g);
      } else {
#pragma unroll
        for (int i = 0; i < kRnElems; ++i) {
          ds[i] = fmaf(dt[i], y[i] * f[i], ds[i]);
          dt[i] *= s[i];
        }
      }
      if (p.post) {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < kRnElems; ++i) {
          dp[i] = fmaf(dt[i], y[i], dp[i]);
          dt[i] *= f[i];
          dot = fmaf(dt[i], y[i], dot);
        }
        dot = row_sum(dot, red) * inv;
#pragma unroll
        for (int i = 0; i < kRnElems; ++i) dt[i] = rs * (dt[i] - y[i] * dot);
      }
      if (p.dy) R::store(p.dy, row * p.D, D, dt);
    }
  }
  // one partial row per (CTA, row slot)
  float* out = p.part + ((long long)blockIdx.x * blockDim.y + threadIdx.y) * 3 * p.D;
#pragma unroll
  for (int j = 0; j < R::J; ++j) {
    const int c = R::col(j);
    if (c >= p.D) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      out[c + i] = dw[j * VEC + i];
      if (FULL) {
        out[p.D + c + i] = dp[j * VEC + i];
        out[2 * p.D + c + i] = ds[j * VEC + i];
      }
    }
  }
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

constexpr int kRnMaxParts = 148 * 8;  // partial rows of the backward

// threads of a row and rows of a CTA
static dim3 rn_block(int D, long long rows) {
  const int tx = ((D + kRnElems - 1) / kRnElems + 31) / 32 * 32;
  int ty = 1;
  while (ty < 8 && tx * ty * 2 <= 256 && rows > ty) ty *= 2;
  return dim3(unsigned(tx), unsigned(ty));
}

static int rn_vec(int D, int es, std::initializer_list<const void*> ptrs,
                  std::initializer_list<long long> strides) {
  int vec = 16 / es;
  for (; vec > 1; vec /= 2) {
    bool ok = D % vec == 0;
    for (const void* q : ptrs) ok = ok && (!q || aligned(q, size_t(vec) * es));
    for (long long st : strides) ok = ok && st % vec == 0;
    if (ok) break;
  }
  // the kernels are built for the full width and for single elements
  return vec == 16 / es ? vec : 1;
}

static int rn_checks(int dtype, long long rows, int D) {
  CYFA_REQUIRE(rows > 0 && rows < (1ll << 31) && D > 0 && D <= kRnMaxWidth, kBadShape);
  CYFA_REQUIRE(dtype == 0 || dtype == 1, kBadDtype);
  return kOk;
}

static unsigned rn_bwd_grid(dim3 block, long long rows) {
  const int per_sm = std::max(1, 1024 / int(block.x * block.y));
  const long long ctas = (rows + block.y - 1) / block.y;
  return unsigned(std::min<long long>({ctas, 148ll * per_sm, (long long)kRnMaxParts / block.y}));
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
  const dim3 block = rn_block(a->D, a->rows);
  const unsigned grid = unsigned((a->rows + block.y - 1) / block.y);
  const int vec = rn_vec(a->D, es, {a->x, a->y, a->gate, xn, h},
                         {a->x_stride, a->y ? a->y_stride : 0, a->gate ? a->gate_stride : 0});
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define CYFA_RN(T, VEC)            \
  CYFA_LAUNCH("residual_norm_fwd", s, \
              (launch_k(residual_norm_fwd_kernel<T, VEC>, grid, block, 0, s, p)))
  if (a->dtype == 1) {
    if (vec == 8) CYFA_RN(__nv_bfloat16, 8); else CYFA_RN(__nv_bfloat16, 1);
  } else {
    if (vec == 4) CYFA_RN(float, 4); else CYFA_RN(float, 1);
  }
#undef CYFA_RN
  return launch_status();
}

size_t cyfa_residual_norm_bwd_work_bytes(long long rows, int D) {
  if (rows <= 0 || D <= 0 || D > kRnMaxWidth) return 0;
  const dim3 block = rn_block(D, rows);
  return size_t(rn_bwd_grid(block, rows)) * block.y * 3 * D * sizeof(float);
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
  const dim3 block = rn_block(a->D, a->rows);
  const unsigned grid = rn_bwd_grid(block, a->rows);
  const int vec = rn_vec(a->D, es, {a->x, a->y, a->gate, dxn, dh, dx, dy, dgate},
                         {a->x_stride, a->y ? a->y_stride : 0, a->gate ? a->gate_stride : 0});
  // without gate, scale and post-norm, dy equals dx: the plain sum's gradient
  const bool full = a->y && (dy || dgate || dpost || dscale);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define CYFA_RN(T, VEC)                                                                        \
  do {                                                                                         \
    if (full)                                                                                  \
      CYFA_LAUNCH("residual_norm_bwd", s,                                                      \
                  (launch_k(residual_norm_bwd_kernel<T, VEC, true>, grid, block, 0, s, p)));   \
    else                                                                                       \
      CYFA_LAUNCH("residual_norm_bwd", s,                                                      \
                  (launch_k(residual_norm_bwd_kernel<T, VEC, false>, grid, block, 0, s, p)));  \
  } while (0)
  if (a->dtype == 1) {
    if (vec == 8) CYFA_RN(__nv_bfloat16, 8); else CYFA_RN(__nv_bfloat16, 1);
  } else {
    if (vec == 4) CYFA_RN(float, 4); else CYFA_RN(float, 1);
  }
#undef CYFA_RN
  if (dweight || dpost || dscale)
    CYFA_LAUNCH("residual_norm_sum", s,
                (launch_k(residual_norm_sum_kernel, dim3(unsigned((a->D + 31) / 32), 3), dim3(32, 32),
                          0, s, p.part, int(grid * block.y), a->D, dweight, dpost, dscale)));
  return launch_status();
}

}  // extern "C"
