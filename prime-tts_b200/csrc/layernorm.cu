// layernorm.cu -- pt_b200_layer_norm and its gradient.
//
//   y  = (x - mean) * rstd * gamma + beta          mean, var over the row; rstd = 1 / sqrt(var + eps)
//   g  = dy * gamma;  xhat = (x - mean) * rstd
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dgamma = sum over rows of dy * xhat;  dbeta = sum over rows of dy
//
// Both passes are bound by HBM: forward reads x and writes y once, backward reads x and dy and
// writes dx once; the row lives in registers between its reduction and its use.  The variance is
// the mean of the squared deviations from the mean already known (two sums over registers, not a
// difference of two large sums).
//
// A row is owned by TPR threads: a warp when it fits the warp's registers (no barriers, the
// reductions are shuffles), else a block of 256.  Rows wider than kMaxRegCols are read again
// instead of kept.  The weight gradients are column sums over all rows: each block keeps its own
// rows' sums in registers, adds its warps' sums in shared memory and writes one row of partials,
// and a second kernel adds the blocks' partials in their order, so that results do not depend on
// timing.
#include "ops.cuh"

using namespace ptb;

namespace {

constexpr int kBlock = 256;
constexpr int kMaxRegCols = 16384;

// Sum of v over the TPR threads of a row (all of them get it).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *red) {
  v = warp_sum(v);
  if constexpr (TPR == 32) return v;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < TPR / 32; ++i) s += red[i];
  __syncthreads();
  return s;
}

// Two sums with one pair of barriers.
template <int TPR>
__device__ __forceinline__ void row_sum2(float &a, float &b, float *red) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (TPR == 32) return;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    red[warp] = a;
    red[8 + warp] = b;
  }
  __syncthreads();
  a = b = 0.0f;
#pragma unroll
  for (int i = 0; i < TPR / 32; ++i) {
    a += red[i];
    b += red[8 + i];
  }
  __syncthreads();
}

struct NormArgs {
  const void *x, *dy, *gamma, *beta;
  void *y;                     // forward: y; backward: dx (may be null)
  float *mean, *rstd;          // forward: written (may be null); backward: read
  float *part;                 // backward: [blocks][2][cols] partial dgamma, dbeta (may be null)
  int64_t rows, cols, ldx, lddy, ldy;
  float eps;
};

// Element j of thread t's vector i sits in column (i * TPR + t) * V + j.
template <class T, int TPR, int V, int N>
__global__ void __launch_bounds__(kBlock) norm_fwd_kernel(const NormArgs a) {
  constexpr int kRows = kBlock / TPR;
  __shared__ float red[16];
  const int t = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(a.cols);
  using P = Pack<T, V>;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR; r < a.rows;
       r += static_cast<int64_t>(gridDim.x) * kRows) {
    const T *x = static_cast<const T *>(a.x) + r * a.ldx;
    float v[N * V], s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < a.cols) {
        const P p = *reinterpret_cast<const P *>(x + c);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[i * V + j] = to_f32(p.v[j]);
          s += v[i * V + j];
        }
      }
    }
    const float mean = row_sum<TPR>(s, red) * inv;
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i * TPR + t) * V < a.cols)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = v[i * V + j] - mean;
          q = fmaf(d, d, q);
        }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(q, red) * inv + a.eps);
    if (t == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
    T *y = static_cast<T *>(a.y) + r * a.ldy;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < a.cols) {
        P g, b, o;
        if (a.gamma) g = *reinterpret_cast<const P *>(static_cast<const T *>(a.gamma) + c);
        if (a.beta) b = *reinterpret_cast<const P *>(static_cast<const T *>(a.beta) + c);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float f = (v[i * V + j] - mean) * rstd;
          if (a.gamma) f *= to_f32(g.v[j]);
          if (a.beta) f += to_f32(b.v[j]);
          o.v[j] = from_f32<T>(f);
        }
        *reinterpret_cast<P *>(y + c) = o;
      }
    }
  }
}

// Rows wider than the registers hold: three passes over the row, which stays in L2.
template <class T>
__global__ void __launch_bounds__(kBlock) norm_fwd_wide_kernel(const NormArgs a) {
  __shared__ float red[16];
  const float inv = 1.0f / static_cast<float>(a.cols);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + r * a.ldx;
    float s = 0.0f, q = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kBlock) s += to_f32(x[c]);
    const float mean = row_sum<kBlock>(s, red) * inv;
    for (int64_t c = threadIdx.x; c < a.cols; c += kBlock) {
      const float d = to_f32(x[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(row_sum<kBlock>(q, red) * inv + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
    T *y = static_cast<T *>(a.y) + r * a.ldy;
    for (int64_t c = threadIdx.x; c < a.cols; c += kBlock) {
      float f = (to_f32(x[c]) - mean) * rstd;
      if (a.gamma) f *= to_f32(static_cast<const T *>(a.gamma)[c]);
      if (a.beta) f += to_f32(static_cast<const T *>(a.beta)[c]);
      y[c] = from_f32<T>(f);
    }
  }
}

template <class T, int TPR, int V, int N>
__global__ void __launch_bounds__(kBlock) norm_bwd_kernel(const NormArgs a) {
  constexpr int kRows = kBlock / TPR;
  __shared__ float red[16];
  extern __shared__ float acc[];          // TPR == 32: [2][cols], the block's column sums
  const int t = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(a.cols);
  using P = Pack<T, V>;
  float dg[N * V], db[N * V];
#pragma unroll
  for (int i = 0; i < N * V; ++i) dg[i] = db[i] = 0.0f;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR; r < a.rows;
       r += static_cast<int64_t>(gridDim.x) * kRows) {
    const T *x = static_cast<const T *>(a.x) + r * a.ldx;
    const T *dy = static_cast<const T *>(a.dy) + r * a.lddy;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float xh[N * V], g[N * V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < a.cols) {
        const P px = *reinterpret_cast<const P *>(x + c);
        const P pd = *reinterpret_cast<const P *>(dy + c);
        P pg;
        if (a.gamma) pg = *reinterpret_cast<const P *>(static_cast<const T *>(a.gamma) + c);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int k = i * V + j;
          const float d = to_f32(pd.v[j]);
          xh[k] = (to_f32(px.v[j]) - mean) * rstd;
          g[k] = a.gamma ? d * to_f32(pg.v[j]) : d;
          s1 += g[k];
          s2 = fmaf(g[k], xh[k], s2);
          dg[k] = fmaf(d, xh[k], dg[k]);
          db[k] += d;
        }
      }
    }
    row_sum2<TPR>(s1, s2, red);
    if (!a.y) continue;
    s1 *= inv;
    s2 *= inv;
    T *dx = static_cast<T *>(a.y) + r * a.ldy;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < a.cols) {
        P o;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int k = i * V + j;
          o.v[j] = from_f32<T>(rstd * (g[k] - s1 - xh[k] * s2));
        }
        *reinterpret_cast<P *>(dx + c) = o;
      }
    }
  }
  if (!a.part) return;
  float *part = a.part + 2 * a.cols * blockIdx.x;
  if constexpr (TPR == 32) {
    // the block's warps add their sums one after another (a fixed order)
    for (int w = 0; w < kRows; ++w) {
      if (static_cast<int>(threadIdx.x >> 5) == w) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = (i * TPR + t) * V;
          if (c < a.cols)
#pragma unroll
            for (int j = 0; j < V; ++j) {
              acc[c + j] = (w ? acc[c + j] : 0.0f) + dg[i * V + j];
              acc[a.cols + c + j] = (w ? acc[a.cols + c + j] : 0.0f) + db[i * V + j];
            }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.cols; c += kBlock) part[c] = acc[c];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < a.cols)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          part[c + j] = dg[i * V + j];
          part[a.cols + c + j] = db[i * V + j];
        }
    }
  }
}

// Wide rows: dx row by row, the column sums by a block per 32 columns (norm_cols_wide_kernel).
template <class T>
__global__ void __launch_bounds__(kBlock) norm_bwd_wide_kernel(const NormArgs a) {
  __shared__ float red[16];
  const float inv = 1.0f / static_cast<float>(a.cols);
  const T *gamma = static_cast<const T *>(a.gamma);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + r * a.ldx;
    const T *dy = static_cast<const T *>(a.dy) + r * a.lddy;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kBlock) {
      const float g = to_f32(dy[c]) * (gamma ? to_f32(gamma[c]) : 1.0f);
      s1 += g;
      s2 = fmaf(g, (to_f32(x[c]) - mean) * rstd, s2);
    }
    row_sum2<kBlock>(s1, s2, red);
    s1 *= inv;
    s2 *= inv;
    T *dx = static_cast<T *>(a.y) + r * a.ldy;
    for (int64_t c = threadIdx.x; c < a.cols; c += kBlock) {
      const float g = to_f32(dy[c]) * (gamma ? to_f32(gamma[c]) : 1.0f);
      dx[c] = from_f32<T>(rstd * (g - s1 - (to_f32(x[c]) - mean) * rstd * s2));
    }
  }
}

// Column sums of wide rows: block b of gridDim.y row ranges, 32 columns x 8 row lanes.
template <class T>
__global__ void __launch_bounds__(kBlock) norm_cols_wide_kernel(const NormArgs a) {
  __shared__ float sg[8][33], sb[8][33];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int lane = threadIdx.x >> 5;
  float dg = 0.0f, db = 0.0f;
  if (c < a.cols)
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + lane; r < a.rows;
         r += static_cast<int64_t>(gridDim.y) * 8) {
      const float d = to_f32(static_cast<const T *>(a.dy)[r * a.lddy + c]);
      dg = fmaf(d, (to_f32(static_cast<const T *>(a.x)[r * a.ldx + c]) - a.mean[r]) * a.rstd[r], dg);
      db += d;
    }
  sg[lane][threadIdx.x & 31] = dg;
  sb[lane][threadIdx.x & 31] = db;
  __syncthreads();
  if (threadIdx.x < 32 && c < a.cols) {
    dg = db = 0.0f;
    for (int i = 0; i < 8; ++i) {
      dg += sg[i][threadIdx.x];
      db += sb[i][threadIdx.x];
    }
    float *part = a.part + 2 * a.cols * blockIdx.y;
    part[c] = dg;
    part[a.cols + c] = db;
  }
}

// [parts][n] -> out[n]: 32 columns x 8 lanes of parts per block, added in a fixed order.
template <class T>
__global__ void __launch_bounds__(kBlock)
    reduce_columns_kernel(const float *__restrict__ part, int parts, int64_t n, T *__restrict__ out,
                          int64_t out_n, T *__restrict__ out2) {
  __shared__ float s[8][33];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int lane = threadIdx.x >> 5;
  float v = 0.0f;
  if (c < n)
    for (int p = lane; p < parts; p += 8) v += part[p * n + c];
  s[lane][threadIdx.x & 31] = v;
  __syncthreads();
  if (threadIdx.x < 32 && c < n) {
    v = 0.0f;
    for (int i = 0; i < 8; ++i) v += s[i][threadIdx.x];
    T *o = c < out_n ? out + c : (out2 ? out2 + (c - out_n) : nullptr);
    if (o && (c >= out_n || out)) *o = from_f32<T>(v);
  }
}

int64_t grid_rows(const pt_b200_ops *h, int64_t rows, int rows_per_block, int per_sm) {
  const int64_t want = (rows + rows_per_block - 1) / rows_per_block;
  const int64_t cap = static_cast<int64_t>(h->sms) * per_sm;
  return want < cap ? want : cap;
}

// Backward blocks: at most this many rows of partials.
constexpr int kBwdPerSm = 4;
int bwd_blocks(const pt_b200_ops *h, int64_t rows, int64_t cols) {
  if (cols > kMaxRegCols) return static_cast<int>(rows < 8 * 64 ? (rows + 7) / 8 : 64);
  return static_cast<int>(grid_rows(h, rows, cols <= 1024 ? kBlock / 32 : 1, kBwdPerSm));
}

// fn.template operator()<TPR, V, N>() for the smallest instance that holds `cols`.
template <class T, bool VEC, class F>
int pick(int64_t cols, F &&fn) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  if (cols <= 1024) {
    const int64_t n = (cols + 32 * V - 1) / (32 * V);
    if (n * V <= 8) return fn.template operator()<32, V, 8 / V>();
    if (n * V <= 16) return fn.template operator()<32, V, 16 / V>();
    return fn.template operator()<32, V, 32 / V>();
  }
  const int64_t n = (cols + 256 * V - 1) / (256 * V);
  if (n * V <= 8) return fn.template operator()<256, V, 8 / V>();
  if (n * V <= 16) return fn.template operator()<256, V, 16 / V>();
  if (n * V <= 32) return fn.template operator()<256, V, 32 / V>();
  return fn.template operator()<256, V, 64 / V>();
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class T, bool VEC>
struct FwdLaunch {
  const pt_b200_ops *h;
  const NormArgs &a;
  cudaStream_t st;
  template <int TPR, int V, int N>
  int operator()() const {
    norm_fwd_kernel<T, TPR, V, N>
        <<<static_cast<unsigned>(grid_rows(h, a.rows, kBlock / TPR, 8)), kBlock, 0, st>>>(a);
    return 0;
  }
};

template <class T, bool VEC>
struct BwdLaunch {
  const pt_b200_ops *h;
  const NormArgs &a;
  cudaStream_t st;
  template <int TPR, int V, int N>
  int operator()() const {
    const size_t smem = TPR == 32 && a.part ? static_cast<size_t>(2 * a.cols) * 4 : 0;
    norm_bwd_kernel<T, TPR, V, N>
        <<<static_cast<unsigned>(bwd_blocks(h, a.rows, a.cols)), kBlock, smem, st>>>(a);
    return 0;
  }
};

}  // namespace

namespace ptb {
template <class T>
int reduce_columns(const float *part, int parts, int64_t n, T *out, cudaStream_t st) {
  reduce_columns_kernel<T><<<static_cast<unsigned>((n + 31) / 32), kBlock, 0, st>>>(part, parts, n, out,
                                                                                   n, nullptr);
  PTB_CUDA(cudaGetLastError());
  count_launch();
  return 0;
}
template int reduce_columns<float>(const float *, int, int64_t, float *, cudaStream_t);
template int reduce_columns<__nv_bfloat16>(const float *, int, int64_t, __nv_bfloat16 *, cudaStream_t);
template int reduce_columns<__half>(const float *, int, int64_t, __half *, cudaStream_t);
}  // namespace ptb

extern "C" int pt_b200_layer_norm(pt_b200_ops *h, void *stream, const pt_b200_norm_args *p) {
  PTB_REQUIRE(h && p, "pt_b200_layer_norm: NULL handle or arguments");
  PTB_REQUIRE(p->dtype >= PT_B200_F32 && p->dtype <= PT_B200_F16, "pt_b200_layer_norm: unknown element type %d",
              p->dtype);
  PTB_REQUIRE(p->rows >= 0 && p->cols > 0 && p->cols <= (int64_t(1) << 30), "pt_b200_layer_norm: rows %lld x cols %lld",
              (long long)p->rows, (long long)p->cols);
  const int eb = dtype_bytes(p->dtype);
  PTB_REQUIRE(rows_ok(p->x, p->rows, p->cols, p->ldx, eb) && rows_ok(p->y, p->rows, p->cols, p->ldy, eb),
              "pt_b200_layer_norm: x and y need a pointer and a row stride of at least cols");
  PTB_REQUIRE(p->eps >= 0.0f, "pt_b200_layer_norm: eps must not be negative");
  if (p->rows == 0) return 0;
  DeviceScope on(h->device);
  PTB_REQUIRE(on.ok, "pt_b200_layer_norm: device %d cannot be used", h->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NormArgs a{};
  a.x = p->x;
  a.gamma = p->gamma;
  a.beta = p->beta;
  a.y = p->y;
  a.mean = p->mean;
  a.rstd = p->rstd;
  a.rows = p->rows;
  a.cols = p->cols;
  a.ldx = p->ldx;
  a.ldy = p->ldy;
  a.eps = p->eps;
  const int v = 16 / eb;
  const bool vec = p->cols % v == 0 && (p->rows == 1 || (p->ldx % v == 0 && p->ldy % v == 0)) &&
                   aligned16(p->x) && aligned16(p->y) && aligned16(p->gamma) && aligned16(p->beta);
  const int rc = with_dtype(p->dtype, [&](auto *z) {
    using T = std::remove_pointer_t<decltype(z)>;
    if (a.cols > kMaxRegCols) {
      norm_fwd_wide_kernel<T><<<static_cast<unsigned>(grid_rows(h, a.rows, 1, 8)), kBlock, 0, st>>>(a);
      return 0;
    }
    return vec ? pick<T, true>(a.cols, FwdLaunch<T, true>{h, a, st})
               : pick<T, false>(a.cols, FwdLaunch<T, false>{h, a, st});
  });
  if (rc) return rc;
  PTB_CUDA(cudaGetLastError());
  count_launch();
  return 0;
}

extern "C" int64_t pt_b200_layer_norm_backward_work(const pt_b200_ops *h, int64_t rows, int64_t cols) {
  if (!h || rows <= 0 || cols <= 0) return 0;
  return static_cast<int64_t>(bwd_blocks(h, rows, cols)) * 2 * cols * 4;
}

extern "C" int pt_b200_layer_norm_backward(pt_b200_ops *h, void *stream,
                                           const pt_b200_norm_grad_args *p) {
  PTB_REQUIRE(h && p, "pt_b200_layer_norm_backward: NULL handle or arguments");
  PTB_REQUIRE(p->dtype >= PT_B200_F32 && p->dtype <= PT_B200_F16,
              "pt_b200_layer_norm_backward: unknown element type %d", p->dtype);
  PTB_REQUIRE(p->rows >= 0 && p->cols > 0 && p->cols <= (int64_t(1) << 30),
              "pt_b200_layer_norm_backward: rows %lld x cols %lld", (long long)p->rows, (long long)p->cols);
  const int eb = dtype_bytes(p->dtype);
  PTB_REQUIRE(rows_ok(p->x, p->rows, p->cols, p->ldx, eb) && rows_ok(p->dy, p->rows, p->cols, p->lddy, eb) &&
                  (!p->dx || rows_ok(p->dx, p->rows, p->cols, p->lddx, eb)),
              "pt_b200_layer_norm_backward: x, dy and dx need a pointer and a row stride of at least cols");
  PTB_REQUIRE(p->rows == 0 || (p->mean && p->rstd), "pt_b200_layer_norm_backward: mean and rstd are needed");
  PTB_REQUIRE(p->rows == 0 || p->dx || p->dgamma || p->dbeta, "pt_b200_layer_norm_backward: nothing to compute");
  DeviceScope on(h->device);
  PTB_REQUIRE(on.ok, "pt_b200_layer_norm_backward: device %d cannot be used", h->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->rows == 0) {   // sums over no rows
    if (p->dgamma) PTB_CUDA(cudaMemsetAsync(p->dgamma, 0, p->cols * eb, st));
    if (p->dbeta) PTB_CUDA(cudaMemsetAsync(p->dbeta, 0, p->cols * eb, st));
    return 0;
  }
  const bool sums = p->dgamma || p->dbeta;
  const int64_t need = sums ? pt_b200_layer_norm_backward_work(h, p->rows, p->cols) : 0;
  PTB_REQUIRE(need == 0 || (p->work && p->work_bytes >= need && aligned16(p->work)),
              "pt_b200_layer_norm_backward: %lld bytes of 16-byte aligned workspace are needed, %lld given",
              (long long)need, (long long)p->work_bytes);
  NormArgs a{};
  a.x = p->x;
  a.dy = p->dy;
  a.gamma = p->gamma;
  a.y = p->dx;
  a.mean = const_cast<float *>(p->mean);
  a.rstd = const_cast<float *>(p->rstd);
  a.part = sums ? static_cast<float *>(p->work) : nullptr;
  a.rows = p->rows;
  a.cols = p->cols;
  a.ldx = p->ldx;
  a.lddy = p->lddy;
  a.ldy = p->lddx;
  const int v = 16 / eb;
  const bool vec = p->cols % v == 0 &&
                   (p->rows == 1 || (p->ldx % v == 0 && p->lddy % v == 0 && (!p->dx || p->lddx % v == 0))) &&
                   aligned16(p->x) && aligned16(p->dy) && aligned16(p->dx) && aligned16(p->gamma);
  return with_dtype(p->dtype, [&](auto *z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    int parts = bwd_blocks(h, a.rows, a.cols);
    if (a.cols > kMaxRegCols) {
      if (a.y) {
        norm_bwd_wide_kernel<T><<<static_cast<unsigned>(grid_rows(h, a.rows, 1, 8)), kBlock, 0, st>>>(a);
        PTB_CUDA(cudaGetLastError());
        count_launch();
      }
      if (sums) {
        norm_cols_wide_kernel<T>
            <<<dim3(static_cast<unsigned>((a.cols + 31) / 32), parts), kBlock, 0, st>>>(a);
        PTB_CUDA(cudaGetLastError());
        count_launch();
      }
    } else {
      if (vec ? pick<T, true>(a.cols, BwdLaunch<T, true>{h, a, st})
              : pick<T, false>(a.cols, BwdLaunch<T, false>{h, a, st}))
        return -1;
      PTB_CUDA(cudaGetLastError());
      count_launch();
    }
    if (!sums) return 0;
    reduce_columns_kernel<T><<<static_cast<unsigned>((2 * a.cols + 31) / 32), kBlock, 0, st>>>(
        a.part, parts, 2 * a.cols, static_cast<T *>(p->dgamma), a.cols, static_cast<T *>(p->dbeta));
    PTB_CUDA(cudaGetLastError());
    count_launch();
    return 0;
  });
}
