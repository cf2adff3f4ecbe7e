// layernorm.cu -- pt_b200_layer_norm and its gradient.
//
//   y  = (x - mean) * rstd * gamma + beta          mean, var over the row; rstd = 1 / sqrt(var + eps)
//   g  = dy * gamma;  xhat = (x - mean) * rstd
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dgamma = sum over rows of dy * xhat;  dbeta = sum over rows of dy
//
// Both passes are bound by HBM: forward reads x and writes y once, backward reads x and dy and
// writes dx once.  What that takes is enough bytes in flight while a row is being reduced: rows
// travel through a ring of kDepth slots in shared memory (asynchronous 16-byte copies), so that the
// next rows are on their way without holding registers.  A row of registers per thread with plain
// loads left 8 warps on an SM and ran 16384 x 4096 bf16 at 2.4 TB/s.  The variance is the mean of
// the squared deviations from the mean already known (two sums over registers, not a difference of
// two large sums).
//
// With that, what bounds a 2-byte row is the instructions for it: a row's two reductions cost each of
// its warps some 120, so a row is owned by as few threads as hold it with 32 elements each (TPR = 32
// to 512; 8 or 16 elements in narrow rows), elements go through the arithmetic in pairs (the packed
// fp32 instructions), and gamma and beta wait in shared memory in their own type.  32768 x 4096 bf16
// with 16 elements on 256 threads and single arithmetic: 127 us.  Rows wider than kMaxRegCols are
// read again instead of kept.
//
// Where rows are aligned a thread reads back only what it copied itself, with no barrier; where they
// are not, the aligned 16-byte pieces that hold the row are copied (the elements beside it are not
// used, and none outside the tensor are read) and every thread picks single elements: 32768 x 1001 bf16
// 44 us against 26 at 1024, which is instructions.  Two neighbours at a time, or whole pieces with the
// row's ends masked, cost as many: 59 and 46 us.
//
// The weight gradients are column sums over all rows: each thread keeps its columns' sums over the
// rows it walks; a block adds its rows' sums in shared memory and writes one row of partials, and a
// second kernel adds the blocks' partials in a fixed order, so that results do not depend on timing.
// Few rows need no second kernel: up to eight blocks in a cluster add up through distributed shared
// memory (64 x 128 fp16: 7.4 us a call, 10.5 with a second launch and a workspace).
#include <cooperative_groups.h>

#include "ops.cuh"
#include "ptx.cuh"

using namespace ptb;

namespace {

constexpr int kBlock = 256;
constexpr int kMaxRegCols = 16384;

// The TPR threads of a row: a barrier, and sums that all of them get.  `red` holds 2 x 16 floats
// that the row's previous sum did not use.
template <int TPR>
__device__ __forceinline__ void row_sync(int group) {
  if constexpr (TPR == 32)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *red, int group) {
  v = warp_sum(v);
  if constexpr (TPR == 32) return v;
  const int warp = (threadIdx.x % TPR) >> 5;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  row_sync<TPR>(group);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < TPR / 32; ++i) s += red[i];
  return s;
}
template <int TPR>
__device__ __forceinline__ void row_sum2(float &a, float &b, float *red, int group) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (TPR == 32) return;
  const int warp = (threadIdx.x % TPR) >> 5;
  if ((threadIdx.x & 31) == 0) {
    red[warp] = a;
    red[16 + warp] = b;
  }
  row_sync<TPR>(group);
  a = b = 0.0f;
#pragma unroll
  for (int i = 0; i < TPR / 32; ++i) {
    a += red[i];
    b += red[16 + i];
  }
}

// 1 / sqrt(v): the hardware's approximation and one step of Newton's iteration, which leaves the
// rounding of its last operations.
__device__ __forceinline__ float inv_sqrt(float v) {
  const float y = rsqrtf(v);
  const float e = fmaf(-v * y, y, 1.0f);
  return isfinite(e) ? fmaf(0.5f * y, e, y) : y;   // (1 / sqrt(0) and of infinity are y itself)
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

struct NormArgs {
  const void *x, *dy, *gamma, *beta;
  void *y;                     // forward: y; backward: dx (may be null)
  float *mean, *rstd;          // forward: written (may be null); backward: read
  float *part;                 // backward: [blocks][2][cols] partial dgamma, dbeta (may be null)
  const void *x_end, *dy_end;  // past the last row
  int64_t rows, cols, ldx, lddy, ldy;
  void *dgamma, *dbeta;        // backward, direct: written by the cluster itself (each may be null)
  bool direct;
  int pitch;                   // bytes of one row in a slot, unaligned rows
  float eps;
};

// How rows are spread over threads: element j of thread t's vector i sits in column
// (i * TPR + t) * V + j; V = 1 where rows are not aligned.  A thread works through its elements in
// units of PAIRS pairs: a vector, or two single elements, of which the second may lie beyond the row
// (it reads as 0).
template <class T_, int TPR_, int V_, int N_, int INPUTS>
struct Lay {
  using T = T_;
  using P = Pack<T, V_>;
  static constexpr int TPR = TPR_, V = V_, N = N_, kElems = N * V;
  static constexpr int kUnits = V == 1 ? N / 2 : N, kPairs = V == 1 ? 1 : V / 2;
  static constexpr int kThreads = TPR > kBlock ? TPR : kBlock, kRows = kThreads / TPR;
  static constexpr int kRowBytes = TPR * kElems * static_cast<int>(sizeof(T));   // padded
  static constexpr int kSlot = kRows * (kRowBytes + (V == 1 ? 48 : 0)) * INPUTS;
  // The blocks of an SM (launch bounds below) share 160 KB of it for their rings.  Forward, as many
  // blocks as leave room for two slots each beside gamma and beta, or one where single elements are
  // picked (8192 x 8192 fp16 46 us; with four blocks, which did not all fit, 65).  More rows ahead
  // than four changed nothing.
  static constexpr int room(int blocks) {
    const int ring = 160 * 1024 / blocks, left = 224 * 1024 / blocks - 3 * 1024 - 2 * kRowBytes;
    return INPUTS == 1 && left < ring ? left : ring;
  }
  static constexpr int per_sm(int most) {
    return most > 1 && room(most) < (V == 1 ? 1 : 2) * kSlot ? per_sm(most - 1) : most;
  }
  static constexpr int kPerSm = INPUTS == 1 ? per_sm(kThreads == kBlock ? (V == 1 ? 3 : 4) : 2) : (kThreads == kBlock ? 2 : 1);
  static constexpr int kFit = room(kPerSm) / kSlot;
  static constexpr int kDepth = kFit > 4 ? 4 : kFit < 1 ? 1 : kFit;
  static constexpr int kBytes = kSlot * kDepth;
  static constexpr int kParam = kRowBytes;                                       // gamma, or beta

  // Starts the copies of row `row` (the TPR threads together) of the tensor [begin, end); `at` is this
  // input's part of a slot.
  static __device__ __forceinline__ void fetch(uint32_t at, const T *row, const void *begin, const void *end,
                                               int cols, int pitch, int t, int group) {
    if constexpr (V > 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * TPR + t) * V;
        if (c < cols) copy16(at + (i * kThreads + threadIdx.x) * 16, row + c);
      }
    } else {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15);
      const uintptr_t hi = reinterpret_cast<uintptr_t>(row + cols);
      const bool inside = lo >= reinterpret_cast<uintptr_t>(begin) && hi + 15 <= reinterpret_cast<uintptr_t>(end);
      for (uintptr_t p = lo + t * 16; p < hi; p += TPR * 16) {
        const uint32_t to = at + group * pitch + static_cast<uint32_t>(p - lo);
        if (inside || (p >= reinterpret_cast<uintptr_t>(row) && p + 16 <= hi)) {
          copy16(to, reinterpret_cast<const void *>(p));
        } else {   // the tensor may begin or end inside this piece
          const T *from = reinterpret_cast<const T *>(p);
          T *slot = static_cast<T *>(__cvta_shared_to_generic(to));
#pragma unroll
          for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i)
            if (from + i >= row && from + i < row + cols) slot[i] = from[i];
        }
      }
    }
  }
  static __device__ __forceinline__ int column(int unit, int t) {
    return V == 1 ? 2 * unit * TPR + t : (unit * TPR + t) * V;
  }
  static __device__ __forceinline__ bool second(int unit, int t, int cols) {
    return V > 1 || column(unit, t) + TPR < cols;
  }
  static __device__ __forceinline__ void split(const P &p, float2 (&o)[kPairs]) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) o[j] = make_float2(to_f32(p.v[2 * j]), to_f32(p.v[2 * j + 1]));
  }
  // A unit of the row in a slot, and of gamma or beta.
  static __device__ __forceinline__ void get(const uint8_t *at, const T *row, int cols, int pitch, int t, int group,
                                             int unit, float2 (&o)[kPairs]) {
    if constexpr (V > 1) {
      split(*reinterpret_cast<const P *>(at + (unit * kThreads + threadIdx.x) * 16), o);
    } else {
      const T *p = reinterpret_cast<const T *>(at + group * pitch + (reinterpret_cast<uintptr_t>(row) & 15));
      at_columns(p, cols, t, unit, o);
    }
  }
  static __device__ __forceinline__ void at_columns(const T *p, int cols, int t, int unit, float2 (&o)[kPairs]) {
    const int c = column(unit, t);
    if constexpr (V > 1)
      split(*reinterpret_cast<const P *>(p + c), o);
    else
      o[0] = make_float2(to_f32(p[c]), second(unit, t, cols) ? to_f32(p[c + TPR]) : 0.0f);
  }
  static __device__ __forceinline__ void put(T *p, int cols, int t, int unit, const float2 (&o)[kPairs]) {
    const int c = column(unit, t);
    if constexpr (V > 1) {
      P q;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) q.v[2 * j] = from_f32<T>(o[j].x), q.v[2 * j + 1] = from_f32<T>(o[j].y);
      *reinterpret_cast<P *>(p + c) = q;
    } else {
      p[c] = from_f32<T>(o[0].x);
      if (second(unit, t, cols)) p[c + TPR] = from_f32<T>(o[0].y);
    }
  }
  // gamma or beta into shared memory, `none` where there is none.
  static __device__ __forceinline__ void param(T *to, const void *from, int cols, float none) {
    for (int c = threadIdx.x; c < cols; c += kThreads)
      to[c] = from ? static_cast<const T *>(from)[c] : from_f32<T>(none);
  }
};

template <class L>
__global__ void __launch_bounds__(L::kThreads, L::kPerSm) norm_fwd_kernel(const NormArgs a) {
  using T = typename L::T;
  constexpr int TPR = L::TPR, V = L::V, D = L::kDepth, U = L::kUnits, Q = L::kPairs;
  extern __shared__ __align__(16) uint8_t ring[];   // [kDepth] rows, gamma, beta
  __shared__ float red_all[L::kRows][2][32];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, cols = static_cast<int>(a.cols);
  float(*red)[32] = red_all[group];
  const float inv = 1.0f / static_cast<float>(cols);
  const uint32_t at = smem_u32(ring);
  T *gamma = reinterpret_cast<T *>(ring + L::kBytes), *beta = reinterpret_cast<T *>(ring + L::kBytes + L::kParam);
  const int64_t step = static_cast<int64_t>(gridDim.x) * L::kRows;
  int64_t r = static_cast<int64_t>(blockIdx.x) * L::kRows + group, ahead = r;
  const T *x = static_cast<const T *>(a.x) + r * a.ldx, *xa = x;     // this row, the row to fetch
  T *y = static_cast<T *>(a.y) + r * a.ldy;
  const int64_t xstep = step * a.ldx, ystep = step * a.ldy;
#pragma unroll
  for (int d = 0; d < D - 1; ++d, ahead += step, xa += xstep) {
    if (ahead < a.rows) L::fetch(at + d * L::kSlot, xa, a.x, a.x_end, cols, a.pitch, t, group);
    copy_commit();
  }
  L::param(gamma, a.gamma, cols, 1.0f);
  L::param(beta, a.beta, cols, 0.0f);
  __syncthreads();
  int slot = 0, fill = D - 1;
  for (; r < a.rows; r += step, ahead += step, x += xstep, xa += xstep, y += ystep) {
    if (ahead < a.rows) L::fetch(at + fill * L::kSlot, xa, a.x, a.x_end, cols, a.pitch, t, group);
    copy_commit();
    copy_wait<D - 1>();
    if constexpr (V == 1) row_sync<TPR>(group);
    float2 v[U][Q], s = both(0.0f);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (L::column(i, t) < cols) {
        L::get(ring + slot * L::kSlot, x, cols, a.pitch, t, group, i, v[i]);
#pragma unroll
        for (int j = 0; j < Q; ++j) s = add2(s, v[i][j]);
      }
    const float mean = row_sum<TPR>(s.x + s.y, red[0], group) * inv;
    float2 q = both(0.0f);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (L::column(i, t) < cols) {
        const float2 shift = make_float2(-mean, L::second(i, t, cols) ? -mean : 0.0f);
#pragma unroll
        for (int j = 0; j < Q; ++j) {
          v[i][j] = add2(v[i][j], shift);
          q = fma2(v[i][j], v[i][j], q);
        }
      }
    const float rstd = inv_sqrt(row_sum<TPR>(q.x + q.y, red[1], group) * inv + a.eps);
    if (t == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (L::column(i, t) < cols) {
        float2 g[Q], b[Q];
        L::at_columns(gamma, cols, t, i, g);
        L::at_columns(beta, cols, t, i, b);
#pragma unroll
        for (int j = 0; j < Q; ++j) g[j] = fma2(mul2(v[i][j], both(rstd)), g[j], b[j]);
        L::put(y, cols, t, i, g);
      }
    // (the slot read above is filled again in the next turn, behind this turn's barriers)
    if constexpr (V == 1 && TPR == 32) __syncwarp();
    slot = slot + 1 == D ? 0 : slot + 1;
    fill = fill + 1 == D ? 0 : fill + 1;
  }
}

// Rows wider than the registers hold: three passes over the row, which stays in L2.
template <class T>
__global__ void __launch_bounds__(kBlock) norm_fwd_wide_kernel(const NormArgs a) {
  __shared__ float red[2][32];
  const float inv = 1.0f / static_cast<float>(a.cols);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + r * a.ldx;
    float s = 0.0f, q = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kBlock) s += to_f32(x[c]);
    const float mean = row_sum<kBlock>(s, red[0], 0) * inv;
    for (int64_t c = threadIdx.x; c < a.cols; c += kBlock) {
      const float d = to_f32(x[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = inv_sqrt(row_sum<kBlock>(q, red[1], 0) * inv + a.eps);
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

template <class L>
__global__ void __launch_bounds__(L::kThreads, L::kPerSm) norm_bwd_kernel(const NormArgs a) {
  using T = typename L::T;
  constexpr int TPR = L::TPR, V = L::V, D = L::kDepth, U = L::kUnits, Q = L::kPairs;
  // 32 elements a thread and their two sums fill the registers: those rows are read from their slot
  // again for dx
  constexpr bool kKeep = L::kElems <= 16;
  extern __shared__ __align__(16) uint8_t ring[];   // [kDepth][x, dy], gamma; in the end [kRows][2][cols] sums
  __shared__ float red_all[L::kRows][2][32];
  let_next_start();
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, cols = static_cast<int>(a.cols);
  float(*red)[32] = red_all[group];
  const float inv = 1.0f / static_cast<float>(cols);
  constexpr int kHalf = L::kSlot / 2;               // dy's part of a slot
  const uint32_t at = smem_u32(ring);
  T *gamma = reinterpret_cast<T *>(ring + L::kBytes);
  float2 dg[U][Q], db[U][Q];
#pragma unroll
  for (int i = 0; i < U; ++i)
#pragma unroll
    for (int j = 0; j < Q; ++j) dg[i][j] = db[i][j] = both(0.0f);
  const int64_t step = static_cast<int64_t>(gridDim.x) * L::kRows;
  int64_t r = static_cast<int64_t>(blockIdx.x) * L::kRows + group, ahead = r;
  const T *x = static_cast<const T *>(a.x) + r * a.ldx, *xa = x;      // this row, the row to fetch
  const T *dy = static_cast<const T *>(a.dy) + r * a.lddy, *da = dy;
  T *dx = static_cast<T *>(a.y) + r * a.ldy;
  const int64_t xstep = step * a.ldx, dstep = step * a.lddy, ystep = step * a.ldy;
  auto fetch = [&](int slot) {
    L::fetch(at + slot * L::kSlot, xa, a.x, a.x_end, cols, a.pitch, t, group);
    L::fetch(at + slot * L::kSlot + kHalf, da, a.dy, a.dy_end, cols, a.pitch, t, group);
  };
#pragma unroll
  for (int d = 0; d < D - 1; ++d, ahead += step, xa += xstep, da += dstep) {
    if (ahead < a.rows) fetch(d);
    copy_commit();
  }
  L::param(gamma, a.gamma, cols, 1.0f);
  __syncthreads();
  int slot = 0, fill = D - 1;
  float next_mean = r < a.rows ? a.mean[r] : 0.0f, next_rstd = r < a.rows ? a.rstd[r] : 0.0f;
  for (int turn = 0; r < a.rows;
       r += step, ahead += step, x += xstep, xa += xstep, dy += dstep, da += dstep, dx += ystep, turn ^= 1) {
    if (ahead < a.rows) fetch(fill);
    copy_commit();
    const float mean = next_mean, rstd = next_rstd;
    if (r + step < a.rows) next_mean = a.mean[r + step], next_rstd = a.rstd[r + step];
    copy_wait<D - 1>();
    if constexpr (V == 1) row_sync<TPR>(group);
    const uint8_t *sx = ring + slot * L::kSlot, *sd = sx + kHalf;
    const float2 shift = both(-mean), scale = both(rstd);
    float2 xh[kKeep ? U : 1][Q], g[kKeep ? U : 1][Q], s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (L::column(i, t) < cols) {
        float2 px[Q], pd[Q], pg[Q];
        L::get(sx, x, cols, a.pitch, t, group, i, px);
        L::get(sd, dy, cols, a.pitch, t, group, i, pd);
        L::at_columns(gamma, cols, t, i, pg);
#pragma unroll
        for (int j = 0; j < Q; ++j) {
          const float2 h = mul2(add2(px[j], shift), scale), e = mul2(pd[j], pg[j]);
          s1 = add2(s1, e);
          s2 = fma2(e, h, s2);
          dg[i][j] = fma2(pd[j], h, dg[i][j]);
          db[i][j] = add2(db[i][j], pd[j]);
          if constexpr (kKeep) xh[i][j] = h, g[i][j] = e;
        }
      }
    float m1 = s1.x + s1.y, m2 = s2.x + s2.y;
    row_sum2<TPR>(m1, m2, red[turn], group);
    if (a.y) {
      const float2 n1 = both(-m1 * inv), n2 = both(-m2 * inv);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (L::column(i, t) < cols) {
          float2 px[Q], pd[Q], pg[Q];
          if constexpr (!kKeep) {
            L::get(sx, x, cols, a.pitch, t, group, i, px);
            L::get(sd, dy, cols, a.pitch, t, group, i, pd);
            L::at_columns(gamma, cols, t, i, pg);
          }
#pragma unroll
          for (int j = 0; j < Q; ++j) {
            float2 h, e;
            if constexpr (kKeep)
              h = xh[i][j], e = g[i][j];
            else
              h = mul2(add2(px[j], shift), scale), e = mul2(pd[j], pg[j]);
            px[j] = mul2(fma2(h, n2, add2(e, n1)), scale);
          }
          L::put(dx, cols, t, i, px);
        }
    }
    // the slot read above is filled again in the next turn
    if constexpr (V == 1 && (TPR == 32 || !kKeep)) row_sync<TPR>(group);
    slot = slot + 1 == D ? 0 : slot + 1;
    fill = fill + 1 == D ? 0 : fill + 1;
  }
  if (!a.part && !a.direct) return;
  float *part = a.part + 2 * a.cols * blockIdx.x;
  auto give = [&](float *to) {   // this row's sums, [2][cols]
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = L::column(i, t);
      if (c < cols) {
        if constexpr (V == 1) {
          to[c] = dg[i][0].x;
          to[cols + c] = db[i][0].x;
          if (L::second(i, t, cols)) to[c + TPR] = dg[i][0].y, to[cols + c + TPR] = db[i][0].y;
        } else {
#pragma unroll
          for (int j = 0; j < Q; j += 2) {
            *reinterpret_cast<float4 *>(to + c + 2 * j) = make_float4(dg[i][j].x, dg[i][j].y, dg[i][j + 1].x, dg[i][j + 1].y);
            *reinterpret_cast<float4 *>(to + cols + c + 2 * j) =
                make_float4(db[i][j].x, db[i][j].y, db[i][j + 1].x, db[i][j + 1].y);
          }
        }
      }
    }
  };
  static_assert(L::kBytes >= L::kRows * 2 * TPR * L::kElems * 4, "the sums need the ring's room");
  if (a.direct) {
    namespace cg = cooperative_groups;
    auto cluster = cg::this_cluster();
    float *acc = reinterpret_cast<float *>(ring);
    copy_wait<0>();
    __syncthreads();
    give(acc + group * 2 * cols);
    __syncthreads();
    if constexpr (L::kRows > 1)
      for (int c = threadIdx.x; c < 2 * cols; c += L::kThreads) {
        float v = acc[c];
#pragma unroll
        for (int w = 1; w < L::kRows; ++w) v += acc[w * 2 * cols + c];
        acc[c] = v;
      }
    cluster.sync();
    const int blocks = static_cast<int>(gridDim.x);
    for (int c = static_cast<int>(blockIdx.x) * L::kThreads + threadIdx.x; c < 2 * cols; c += blocks * L::kThreads) {
      float v = 0.0f;
      for (int b = 0; b < blocks; ++b) v += cluster.map_shared_rank(acc, b)[c];
      T *out = c < cols ? static_cast<T *>(a.dgamma) : static_cast<T *>(a.dbeta);
      if (out) out[c < cols ? c : c - cols] = from_f32<T>(v);
    }
    cluster.sync();   // no block leaves while another still reads its sums
  } else if constexpr (L::kRows == 1) {
    give(part);
  } else {   // the block's rows meet in the ring, whose copies have all been used, and are added in order
    float *acc = reinterpret_cast<float *>(ring);
    copy_wait<0>();
    __syncthreads();
    give(acc + group * 2 * cols);
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * cols; c += L::kThreads) {
      float v = acc[c];
#pragma unroll
      for (int w = 1; w < L::kRows; ++w) v += acc[w * 2 * cols + c];
      part[c] = v;
    }
  }
}

// Wide rows: dx row by row, the column sums by a block per 32 columns (norm_cols_wide_kernel).
template <class T>
__global__ void __launch_bounds__(kBlock) norm_bwd_wide_kernel(const NormArgs a) {
  __shared__ float red[2][32];
  int turn = 0;
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
    row_sum2<kBlock>(s1, s2, red[turn], 0);
    turn ^= 1;
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

// [parts][n] -> out[n] (and out2 from out_n on): 32 columns x LANES per block; a lane adds every
// LANES-th partial (lane_sum), then the lanes are added in order.
template <class T, int LANES>
__global__ void __launch_bounds__(32 * LANES)
    reduce_columns_kernel(const float *__restrict__ part, int parts, int64_t n, T *__restrict__ out,
                          int64_t out_n, T *__restrict__ out2) {
  __shared__ float s[LANES][33];
  wait_for_previous();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int lane = threadIdx.x >> 5;
  float v = 0.0f;
  if (c < n) v = lane_sum(part + c, lane, parts, LANES, n);
  s[lane][threadIdx.x & 31] = v;
  __syncthreads();
  if (threadIdx.x < 32 && c < n) {
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < LANES; ++i) v += s[i][threadIdx.x];
    if (c < out_n) {
      if (out) out[c] = from_f32<T>(v);
    } else if (out2) {
      out2[c - out_n] = from_f32<T>(v);
    }
  }
}

// Launched so that it may start while the kernel that writes the partials still runs.
template <class T, int LANES>
int launch_reduce(const float *part, int parts, int64_t n, T *out, int64_t out_n, T *out2, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((n + 31) / 32));
  cfg.blockDim = dim3(32 * LANES);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  PTB_CUDA(cudaLaunchKernelEx(&cfg, reduce_columns_kernel<T, LANES>, part, parts, n, out, out_n, out2));
  count_launch();
  return 0;
}

int64_t grid_rows(const pt_b200_ops *h, int64_t rows, int rows_per_block, int per_sm) {
  const int64_t want = (rows + rows_per_block - 1) / rows_per_block;
  const int64_t cap = static_cast<int64_t>(h->sms) * per_sm;
  return want < cap ? want : cap;
}

// fn.template operator()<TPR, V, N>() for the threads and elements of a row.  Few elements a thread
// where there are too few rows to fill the GPU (`few`), where one row's latency counts: 64 x 4096 fp32
// backward took 10.3 us with 32 elements and 7.7 with 16.  Single elements: 16 a thread, which need no
// more than their registers (32768 x 1001 fp32 47 us, with 32 elements 64).  Backward, rows of up to 2048 keep 8 or 16
// elements, whose sums leave room for more rows at once (8192 x 1000 fp16 16 us, with 32 elements 32);
// rows of up to 8192 take 32 on 256 threads, two blocks an SM (4000 x 6144 bf16 40 us, with 16 on 512 46).
template <class T, bool VEC, bool FORWARD, class F>
int pick(int64_t cols, bool few, F &&fn) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  if (cols <= 256) return fn.template operator()<32, V, 8 / V>();
  if (cols <= 512) return fn.template operator()<32, V, 16 / V>();
  if (cols <= 1024 && (few || !FORWARD)) return fn.template operator()<128, V, 8 / V>();
  if (cols <= 4096 && few) return fn.template operator()<512, V, 8 / V>();
  if (cols <= 8192 && few && cols > 4096) return fn.template operator()<512, V, 16 / V>();
  if constexpr (FORWARD && !VEC) {
    if (cols <= 1024) return fn.template operator()<64, V, 16 / V>();
    if (cols <= 2048) return fn.template operator()<128, V, 16 / V>();
    if (cols <= 4096) return fn.template operator()<256, V, 16 / V>();
    if (cols <= 8192) return fn.template operator()<512, V, 16 / V>();
  } else if constexpr (FORWARD) {
    if (cols <= 1024) return fn.template operator()<32, V, 32 / V>();
    if (cols <= 2048) return fn.template operator()<64, V, 32 / V>();
    if (cols <= 8192 && cols > 4096) return fn.template operator()<256, V, 32 / V>();
  } else {
    if (cols <= 2048) return fn.template operator()<128, V, 16 / V>();
    if (cols <= 8192 && cols > 4096) return fn.template operator()<256, V, 32 / V>();
  }
  if (cols <= 4096) return fn.template operator()<128, V, 32 / V>();
  return fn.template operator()<512, V, 32 / V>();
}
bool few_rows(const pt_b200_ops *h, int64_t rows) { return rows < 4 * h->sms; }

int rows_per_block(const pt_b200_ops *h, int64_t rows, int64_t cols) {
  return cols <= 512 ? 8 : cols <= 1024 || (cols <= 4096 && !few_rows(h, rows)) ? 2 : 1;
}
// Backward blocks, which is the number of rows of partials: as many as run at once (two of 256
// threads on an SM, one of 512).
int bwd_blocks(const pt_b200_ops *h, int64_t rows, int64_t cols) {
  if (cols > kMaxRegCols) return static_cast<int>(rows < 8 * 64 ? (rows + 7) / 8 : 64);
  return static_cast<int>(
      grid_rows(h, rows, rows_per_block(h, rows, cols), cols <= 1024 || (cols <= 8192 && !few_rows(h, rows)) ? 2 : 1));
}
// Blocks of the cluster that does a few rows alone (two turns each), or 0.
int direct_blocks(const pt_b200_ops *h, int64_t rows, int64_t cols) {
  if (cols > kMaxRegCols) return 0;
  const int64_t each = 2 * rows_per_block(h, rows, cols);
  for (int n = 1; n <= 8; n *= 2)
    if (rows <= n * each) return n;
  return 0;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Shared memory beyond 48 KB has to be allowed once per kernel and device; it is set at every launch
// that needs it, which costs nothing next to the launch.
template <class K>
int launch_rows(K kernel, int64_t blocks, int threads, size_t smem, const NormArgs &a, cudaStream_t st) {
  if (smem > 40 * 1024)   // (beside the static part, within the 48 KB that need no permission)
    PTB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  kernel<<<static_cast<unsigned>(blocks), threads, smem, st>>>(a);
  PTB_CUDA(cudaGetLastError());
  count_launch();
  return 0;
}

template <class T>
struct FwdLaunch {
  const pt_b200_ops *h;
  const NormArgs &a;
  cudaStream_t st;
  template <int TPR, int V, int N>
  int operator()() const {
    using L = Lay<T, TPR, V, N, 1>;
    return launch_rows(norm_fwd_kernel<L>, grid_rows(h, a.rows, L::kRows, L::kPerSm), L::kThreads,
                       L::kBytes + 2 * L::kParam, a, st);
  }
};

template <class T>
struct BwdLaunch {
  const pt_b200_ops *h;
  const NormArgs &a;
  cudaStream_t st;
  template <int TPR, int V, int N>
  int operator()() const {
    using L = Lay<T, TPR, V, N, 2>;
    if (!a.direct)
      return launch_rows(norm_bwd_kernel<L>, bwd_blocks(h, a.rows, a.cols), L::kThreads, L::kBytes + L::kParam, a, st);
    if (L::kBytes + L::kParam > 40 * 1024)
      PTB_CUDA(cudaFuncSetAttribute(norm_bwd_kernel<L>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    L::kBytes + L::kParam));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(direct_blocks(h, a.rows, a.cols));
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kBytes + L::kParam;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cfg.gridDim.x;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    PTB_CUDA(cudaLaunchKernelEx(&cfg, norm_bwd_kernel<L>, a));
    count_launch();
    return 0;
  }
};

}  // namespace

namespace ptb {
template <class T>
int reduce_columns(const float *part, int parts, int64_t n, T *out, cudaStream_t st) {
  return launch_reduce<T, 8>(part, parts, n, out, n, nullptr, st);
}
template int reduce_columns<float>(const float *, int, int64_t, float *, cudaStream_t);
template int reduce_columns<__nv_bfloat16>(const float *, int, int64_t, __nv_bfloat16 *, cudaStream_t);
template int reduce_columns<__half>(const float *, int, int64_t, __half *, cudaStream_t);
}  // namespace ptb

extern "C" int pt_b200_layer_norm(pt_b200_ops *h, void *stream, const pt_b200_norm_args *p) {
  PTB_REQUIRE(h && p, "pt_b200_layer_norm: NULL handle or arguments");
  PTB_REQUIRE(p->dtype >= PT_B200_F32 && p->dtype <= PT_B200_F16, "pt_b200_layer_norm: unknown element type %d",
              p->dtype);
  PTB_REQUIRE(p->rows >= 0 && p->rows < (int64_t(1) << 31) && p->cols > 0 && p->cols <= (int64_t(1) << 30),
              "pt_b200_layer_norm: rows %lld x cols %lld",
              (long long)p->rows, (long long)p->cols);
  const int eb = dtype_bytes(p->dtype);
  PTB_REQUIRE(rows_ok(p->x, p->rows, p->cols, p->ldx, eb) && rows_ok(p->y, p->rows, p->cols, p->ldy, eb),
              "pt_b200_layer_norm: x and y need an aligned pointer and a row stride of at least cols");
  PTB_REQUIRE(element_ok(p->gamma, eb) && element_ok(p->beta, eb) && element_ok(p->mean, 4) && element_ok(p->rstd, 4),
              "pt_b200_layer_norm: gamma, beta, mean or rstd is not aligned to its elements");
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
  a.x_end = static_cast<const char *>(p->x) + ((p->rows - 1) * p->ldx + p->cols) * eb;
  a.pitch = static_cast<int>(round_up(p->cols * eb, 16) + 32);
  const int v = 16 / eb;
  const bool vec = p->cols % v == 0 && (p->rows == 1 || (p->ldx % v == 0 && p->ldy % v == 0)) &&
                   aligned16(p->x) && aligned16(p->y) && aligned16(p->gamma) && aligned16(p->beta);
  return with_dtype(p->dtype, [&](auto *z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    if (a.cols > kMaxRegCols)
      return launch_rows(norm_fwd_wide_kernel<T>, grid_rows(h, a.rows, 1, 8), kBlock, 0, a, st);
    const bool few = few_rows(h, a.rows);
    return vec ? pick<T, true, true>(a.cols, few, FwdLaunch<T>{h, a, st})
               : pick<T, false, true>(a.cols, few, FwdLaunch<T>{h, a, st});
  });
}

extern "C" int64_t pt_b200_layer_norm_backward_work(const pt_b200_ops *h, int64_t rows, int64_t cols) {
  if (!h || rows <= 0 || cols <= 0 || direct_blocks(h, rows, cols)) return 0;
  return static_cast<int64_t>(bwd_blocks(h, rows, cols)) * 2 * cols * 4;
}

extern "C" int pt_b200_layer_norm_backward(pt_b200_ops *h, void *stream,
                                           const pt_b200_norm_grad_args *p) {
  PTB_REQUIRE(h && p, "pt_b200_layer_norm_backward: NULL handle or arguments");
  PTB_REQUIRE(p->dtype >= PT_B200_F32 && p->dtype <= PT_B200_F16,
              "pt_b200_layer_norm_backward: unknown element type %d", p->dtype);
  PTB_REQUIRE(p->rows >= 0 && p->rows < (int64_t(1) << 31) && p->cols > 0 && p->cols <= (int64_t(1) << 30),
              "pt_b200_layer_norm_backward: rows %lld x cols %lld", (long long)p->rows, (long long)p->cols);
  const int eb = dtype_bytes(p->dtype);
  PTB_REQUIRE(rows_ok(p->x, p->rows, p->cols, p->ldx, eb) && rows_ok(p->dy, p->rows, p->cols, p->lddy, eb) &&
                  (!p->dx || rows_ok(p->dx, p->rows, p->cols, p->lddx, eb)),
              "pt_b200_layer_norm_backward: x, dy and dx need an aligned pointer and a row stride of at least cols");
  PTB_REQUIRE(element_ok(p->gamma, eb) && element_ok(p->mean, 4) && element_ok(p->rstd, 4) &&
                  element_ok(p->dgamma, eb) && element_ok(p->dbeta, eb),
              "pt_b200_layer_norm_backward: gamma, mean, rstd, dgamma or dbeta is not aligned to its elements");
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
  a.direct = sums && direct_blocks(h, p->rows, p->cols);
  a.dgamma = p->dgamma;
  a.dbeta = p->dbeta;
  a.part = sums && !a.direct ? static_cast<float *>(p->work) : nullptr;
  a.rows = p->rows;
  a.cols = p->cols;
  a.ldx = p->ldx;
  a.lddy = p->lddy;
  a.dy_end = static_cast<const char *>(p->dy) + ((p->rows - 1) * p->lddy + p->cols) * eb;
  a.ldy = p->lddx;
  a.x_end = static_cast<const char *>(p->x) + ((p->rows - 1) * p->ldx + p->cols) * eb;
  a.pitch = static_cast<int>(round_up(p->cols * eb, 16) + 32);
  const int v = 16 / eb;
  const bool vec = p->cols % v == 0 &&
                   (p->rows == 1 || (p->ldx % v == 0 && p->lddy % v == 0 && (!p->dx || p->lddx % v == 0))) &&
                   aligned16(p->x) && aligned16(p->dy) && aligned16(p->dx) && aligned16(p->gamma);
  return with_dtype(p->dtype, [&](auto *z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    int parts = bwd_blocks(h, a.rows, a.cols);
    if (a.cols > kMaxRegCols) {
      if (sums) {   // before dx, which may lie over dy
        norm_cols_wide_kernel<T>
            <<<dim3(static_cast<unsigned>((a.cols + 31) / 32), parts), kBlock, 0, st>>>(a);
        PTB_CUDA(cudaGetLastError());
        count_launch();
      }
      if (a.y && launch_rows(norm_bwd_wide_kernel<T>, grid_rows(h, a.rows, 1, 8), kBlock, 0, a, st)) return -1;
    } else if (vec ? pick<T, true, false>(a.cols, few_rows(h, a.rows), BwdLaunch<T>{h, a, st})
                   : pick<T, false, false>(a.cols, few_rows(h, a.rows), BwdLaunch<T>{h, a, st})) {
      return -1;
    }
    if (!sums || a.direct) return 0;
    return launch_reduce<T, 32>(a.part, parts, 2 * a.cols, static_cast<T *>(p->dgamma), a.cols,
                                static_cast<T *>(p->dbeta), st);
  });
}
