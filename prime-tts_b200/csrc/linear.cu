// linear.cu -- pt_b200_linear and its gradient.
//
//   pre = x W^T + b;  y = act(pre) + r
//   dpre = dy * act'(pre);  dx = dpre W;  dW = dpre^T x;  db = sum over rows of dpre
//
// The three products run on the tensor cores (linear_tc.cu); x W^T of a few rows, and of fp32 rows against
// a few channels, in kernels of their own.
#include <algorithm>
#include <type_traits>

#include "linear_tc.cuh"

using namespace ptb;

namespace {

struct FewArgs {
  const void *x, *w;
  int64_t in, out, ldx, ldw;
  int rows, shares;     // shares: warps that split a channel's k
  LinearEpi e;
};

// ---- a few rows (single tokens): every weight is read once and used for all of them, so the call is
// bound by the weights' bytes, and by its latency where they are few.  A warp takes two channels (four
// where there are many rows, which halves what it reads of x) and a share of k: it reads 16 bytes of
// each weight row and of each row of x (which stays in L1) per lane and step, kAhead steps in flight
// with no branch between the loads, and adds up in fp32 FMAs.  Lanes, then the warps that share a
// channel's k, add up in a fixed order.  More rows than eight are groups of eight, which read the
// weights again from L2.  1 x 4096 x 4096 bf16 5.8 us (5.8 TB/s), 8 x 4096 x 4096 fp32 15.6 us; with
// twice as many warps, in two waves, 6.9 and 22.9.
constexpr int kFewGroup = 8, kFewWarps = 8, kFewFill = 8;

// Sums of v[0 .. N) over the warp, by halves: N / 2 + N / 4 + ... exchanges, not 5 N.  Lane l holds
// the sum of value (l / (32 / N)).
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N], int lane) {
  int o = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2, o /= 2) {
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const bool up = lane & o;
      const float give = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  for (; o; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

template <class T, int R, int C, bool VEC>
__global__ void __launch_bounds__(kFewWarps * 32, 2) linear_few_kernel(const FewArgs a) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1, kAhead = VEC ? (R <= 2 ? 4 : R == 4 ? 2 : 1) : 4;
  constexpr int kSums = C * R;
  using P = Pack<T, V>;
  __shared__ float part[kFewWarps][kSums];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = warp % a.shares, team = warp / a.shares;
  const int row0 = blockIdx.y * kFewGroup, rows = min(a.rows - row0, kFewGroup);
  const int64_t chan = (static_cast<int64_t>(blockIdx.x) * (kFewWarps / a.shares) + team) * C;
  float acc[kSums];
#pragma unroll
  for (int i = 0; i < kSums; ++i) acc[i] = 0.0f;
  if (chan < a.out) {
    const int64_t step = static_cast<int64_t>(a.shares) * 32 * V;
    int64_t k = (share * 32 + lane) * V;
    const T *w[C], *x[R];
#pragma unroll
    for (int c = 0; c < C; ++c)   // (the last channel again in the place of one beyond)
      w[c] = static_cast<const T *>(a.w) + (chan + c < a.out ? chan + c : a.out - 1) * a.ldw + k;
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = static_cast<const T *>(a.x) + (row0 + (r < rows ? r : 0)) * a.ldx + k;
    auto steps = [&](auto count) {
      constexpr int A = decltype(count)::value;
      P p[A][C], q[A][R];
#pragma unroll
      for (int u = 0; u < A; ++u) {
#pragma unroll
        for (int c = 0; c < C; ++c) p[u][c] = *reinterpret_cast<const P *>(w[c] + u * step);
#pragma unroll
        for (int r = 0; r < R; ++r) q[u][r] = *reinterpret_cast<const P *>(x[r] + u * step);
      }
#pragma unroll
      for (int u = 0; u < A; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c)
              acc[c * R + r] = fmaf(to_f32(p[u][c].v[j]), to_f32(q[u][r].v[j]), acc[c * R + r]);
#pragma unroll
      for (int c = 0; c < C; ++c) w[c] += A * step;
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] += A * step;
      k += A * step;
    };
    while (k + (kAhead - 1) * step < a.in) steps(std::integral_constant<int, kAhead>{});
    while (k < a.in) steps(std::integral_constant<int, 1>{});
  }
  __syncwarp();
  const float v = warp_sums(acc, lane);
  if (lane % (32 / kSums) == 0) part[warp][lane / (32 / kSums)] = v;
  __syncthreads();
  if (share == 0 && lane < kSums) {
    const int c = lane / R, r = lane % R;
    if (chan + c < a.out && r < rows) {
      float t = 0.0f;
      for (int s = 0; s < a.shares; ++s) t += part[warp + s][lane];
      linear_store<T>(a.e, row0 + r, chan + c, t);
    }
  }
}

template <class T, bool VEC>
int launch_few(const pt_b200_ops *h, const FewArgs &args, cudaStream_t st) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  FewArgs a = args;
  // share a channel's k among warps until there are kFewFill on every SM, or a share is a single step
  const int64_t groups = (a.rows + kFewGroup - 1) / kFewGroup;
  // four channels a warp halve what it reads of x, where there is work for all warps even so
  const bool four = a.rows > 4 && groups * ((a.out + 3) / 4) >= kFewFill * h->sms;
  const int64_t teams = four ? (a.out + 3) / 4 : (a.out + 1) / 2;
  a.shares = 1;
  while (a.shares < kFewWarps && teams * groups * a.shares < kFewFill * h->sms && a.in > a.shares * 32 * V) a.shares *= 2;
  const int64_t per_block = kFewWarps / a.shares;
  const unsigned blocks = static_cast<unsigned>((teams + per_block - 1) / per_block);
  auto *kernel = a.rows == 1 ? linear_few_kernel<T, 1, 2, VEC>
                 : a.rows == 2 ? linear_few_kernel<T, 2, 2, VEC>
                 : a.rows <= 4 ? linear_few_kernel<T, 4, 2, VEC>
                 : four ? linear_few_kernel<T, 8, 4, VEC> : linear_few_kernel<T, 8, 2, VEC>;
  kernel<<<dim3(blocks, static_cast<unsigned>(groups)), kFewWarps * 32, 0, st>>>(a);
  PTB_CUDA(cudaGetLastError());
  count_launch();
  return 0;
}

// ---- fp32, many rows and up to 32 channels: the tensor cores would need planes of all of x, which is
// most of what such a call moves, for products that are a fraction of it.  Here x and the weights go
// through a ring of kNarrowStages steps of 64 of k in shared memory (asynchronous copies, zeros beyond
// the matrices) and the sums are packed fp32 FMAs over pairs of k: a block has 64 rows and all
// channels, a thread four rows (16 apart) and C channels (8 apart), and two groups of threads half of
// each step's k.  Pieces of 16 bytes sit at their place XOR their row, so that neither reads collide.
// Two blocks an SM keep the FMA pipe half busy, next to shared memory's reads.  16384 x 4096 x 32
// 131 us (few rows 238), 15434 x 1592 x 25 55 (81), 16000 x 1592 x 4 30 (73), 16000 x 100 x 20 7.7 (17);
// eight rows a thread and a quarter of k, which reads less: 133, 57, 28, 9.4.
constexpr int kNarrowRows = 64, kNarrowK = 64, kNarrowStages = 3, kNarrowBlock = 256, kNarrowMost = 32;

template <int C, bool VEC>
__global__ void __launch_bounds__(kNarrowBlock, 2) linear_narrow_kernel(const FewArgs a) {
  constexpr int kStage = (kNarrowRows + 8 * C) * kNarrowK;   // floats
  constexpr int kXCopies = kNarrowRows / 16, kWCopies = (8 * C + 15) / 16;
  extern __shared__ __align__(128) float ring_f[];           // [stages][64 rows of x, 8 C of w][64 of k]
  const int tid = threadIdx.x, group = tid >> 7, tx = tid & 7, ty = tid >> 3 & 15;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kNarrowRows;
  // copies: piece `piece` of rows line, line + 16, ...
  const int piece = tid & 15, line = tid >> 4;
  const uint32_t to = smem_u32(ring_f) + (line * kNarrowK + ((piece ^ (line & 7)) << 2)) * 4;
  const float *x = static_cast<const float *>(a.x), *w = static_cast<const float *>(a.w);
  const int steps = static_cast<int>((a.in + kNarrowK - 1) / kNarrowK);
  auto copy = [&](uint32_t dst, const float *base, int64_t row, int64_t rows, int64_t ld, int64_t k) {
    if constexpr (VEC) {
      const bool in = row < rows && k < a.in;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(in ? base + row * ld + k : base),
                   "r"(in ? 16 : 0)
                   : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = row < rows && k + i < a.in;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * i),
                     "l"(in ? base + row * ld + k + i : base), "r"(in ? 4 : 0)
                     : "memory");
      }
    }
  };
  auto fetch = [&](int step) {
    if (step < steps) {
      const uint32_t at = to + step % kNarrowStages * (kStage * 4);
      const int64_t k = static_cast<int64_t>(step) * kNarrowK + piece * 4;
#pragma unroll
      for (int i = 0; i < kXCopies; ++i) copy(at + i * 16 * kNarrowK * 4, x, row0 + line + 16 * i, a.rows, a.ldx, k);
#pragma unroll
      for (int i = 0; i < kWCopies; ++i)
        if (line + 16 * i < 8 * C)
          copy(at + (kNarrowRows + i * 16) * kNarrowK * 4, w, line + 16 * i, a.out, a.ldw, k);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float2 acc[4][C];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) acc[i][j] = both(0.0f);
#pragma unroll
  for (int s = 0; s < kNarrowStages - 1; ++s) fetch(s);
  for (int s = 0; s < steps; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kNarrowStages - 2) : "memory");
    __syncthreads();   // step s has arrived, and the slot of step s - 1 has been read
    fetch(s + kNarrowStages - 1);
    const float *xs = ring_f + s % kNarrowStages * kStage, *ws = xs + kNarrowRows * kNarrowK;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int at = group * 8 + c;
      float4 p[4], q[C];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = *reinterpret_cast<const float4 *>(xs + (ty + 16 * i) * kNarrowK + ((at ^ (ty & 7)) << 2));
#pragma unroll
      for (int j = 0; j < C; ++j)
        q[j] = *reinterpret_cast<const float4 *>(ws + (tx + 8 * j) * kNarrowK + ((at ^ tx) << 2));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          acc[i][j] = fma2(make_float2(p[i].x, p[i].y), make_float2(q[j].x, q[j].y), acc[i][j]);
          acc[i][j] = fma2(make_float2(p[i].z, p[i].w), make_float2(q[j].z, q[j].w), acc[i][j]);
        }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float *other = ring_f + (tid & 127);   // the second group's sums, [4 C][128]
  if (group == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) other[(i * C + j) * 128] = acc[i][j].x + acc[i][j].y;
  }
  __syncthreads();
  if (group == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int64_t row = row0 + ty + 16 * i;
        const int chan = tx + 8 * j;
        if (row < a.rows && chan < a.out)
          linear_store<float>(a.e, row, chan, acc[i][j].x + acc[i][j].y + other[(i * C + j) * 128]);
      }
  }
}

template <int C>
int launch_narrow(const FewArgs &a, bool vec, cudaStream_t st) {
  constexpr int kBytes = kNarrowStages * (kNarrowRows + 8 * C) * kNarrowK * 4;
  auto *kernel = vec ? linear_narrow_kernel<C, true> : linear_narrow_kernel<C, false>;
  PTB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
  kernel<<<static_cast<unsigned>((a.rows + kNarrowRows - 1) / kNarrowRows), kNarrowBlock, kBytes, st>>>(a);
  PTB_CUDA(cudaGetLastError());
  count_launch();
  return 0;
}

// An operand: the tensor itself where the tensor cores can read it, else its planes in the
// workspace, which a pass of `jobs` fills.
int64_t operand_bytes(int dtype, const void *p, int64_t rows, int64_t cols, int64_t ld) {
  return tc_direct(dtype, p, rows, ld) ? 0 : tc_plane_bytes(dtype, rows, cols);
}
TcOperand operand(const pt_b200_ops *h, int dtype, const void *p, int64_t rows, int64_t cols, int64_t ld,
                  char **work, PrepJobs *jobs, int *n) {
  if (tc_direct(dtype, p, rows, ld)) return tc_tensor(p, rows, cols, ld);
  const TcOperand o = tc_planes(*work, rows, cols);
  *work += tc_plane_bytes(dtype, rows, cols);
  PrepJob j{};
  j.src = p;
  j.dst = const_cast<void *>(o.p);
  j.rows = rows;
  j.cols = cols;
  j.ld = ld;
  j.ldd = o.ld;
  j.plane = o.plane;
  tc_add_job(h, dtype, jobs, n, j);
  return o;
}

bool sizes_ok(int64_t rows, int64_t n_in, int64_t n_out) {
  return rows >= 0 && n_in > 0 && n_out > 0 && rows < (int64_t(1) << 31) && n_in < (int64_t(1) << 30) &&
         n_out < (int64_t(1) << 30);
}

// Whether x and w can be read 16 bytes at a time.
bool copies_whole(const pt_b200_linear_args *p) {
  const int v = 16 / dtype_bytes(p->dtype);
  auto aligned = [&](const void *q, int64_t rows, int64_t ld) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (rows == 1 || ld % v == 0);
  };
  return p->in % v == 0 && aligned(p->x, p->rows, p->ldx) && aligned(p->w, p->out, p->ldw);
}

// The kernel that a call takes: by the microseconds that each would take.  The few-rows kernel's follow
// from its warps' tasks (two channels x eight rows), each a start and k; the tensor cores' from a start,
// the first stages of k, the weights and x (in its planes, against a tile of 128 channels).  Fits to
// measurements (the tensor cores' in brackets, rows x in x out):
//   bf16  4 x 4096 x 1024 4.5 (6.8), 8 x 1024 x 1024 3.9 (5.9), 2 x 4096 x 4096 7.4 (8.8), 4 x 4096 x
//         4096 10.5 (8.8), 64 x 192 x 768 5.7 (4.9), 1000 x 64 x 64 6.2 (4.5)
//   not aligned, so that the tensor cores need copies: 128 x 101 x 201 4.4 (5.9), 500 x 101 x 201 10.1
//         (5.9), 4 x 4001 x 4001 16.3 (21), 8 x 4001 x 4001 25.6 (21)
//   fp32, which the tensor cores need in planes: 8 x 4096 x 4096 15.6 (48), 16 x 192 x 768 3.2 (8.7),
//         128 x 768 x 192 5.3 (9.9), 2000 x 192 x 16 3.3 (9.4), 700 x 192 x 192 7.4 (9.1), 7369 x
//         2296 x 24 46 (68), 16064 x 347 x 40 (27)
// The few-rows kernel waits for an x that does not stay in L2.  The narrow one takes a start and, for each
// 64 rows on an SM, steps of k: 1000 x 4096 x 32 73 us (few rows 15.5), 4000 x 1024 x 16 15 (10.5), 2000 x
// 192 x 16 5.5 (3.3), 7369 x 2296 x 24 45 (46), 19434 x 192 x 32 13.9 (tensor cores 19.9).
enum class Way { kTensor, kFew, kNarrow };
constexpr int kFewRows = 1 << 18;
Way way(const pt_b200_ops *h, const pt_b200_linear_args *p) {
  const bool f32 = p->dtype == PT_B200_F32;
  const bool direct = tc_direct(p->dtype, p->x, p->rows, p->ldx) && tc_direct(p->dtype, p->w, p->out, p->ldw);
  const double k = static_cast<double>(p->in), w = k * static_cast<double>(p->out) * 1e-6;
  const double tasks = static_cast<double>((p->rows + kFewGroup - 1) / kFewGroup) * ((p->out + 1) / 2) * 1e-3;
  const double fill = p->rows <= 1 ? 0.125 : p->rows <= 2 ? 0.25 : p->rows <= 4 ? 0.5 : 1.0;   // rows a task has
  const double four = p->rows > 4 && tasks > 2.4 ? 0.7 : 1.0;   // many tasks, of four channels each
  const double start = 0.001 * (k < 1024 ? k : 1024), x = static_cast<double>(p->rows) * k * 1e-6;
  const double wait = f32 && x > 8 ? 1.6 * (x - 8) : 0.0;
  const double few = 2.4 + wait + four * tasks * (0.7 + fill * k * (f32 ? 0.0014 : direct ? 0.0018 : 0.003));
  const double tensor =
      start + (f32 ? 7.6 + 2.4 * w + 4.0 * x : direct ? 4.6 + 0.18 * w + 0.6 * x : 5.7 + 0.9 * w + 1.4 * x);
  if (f32 && p->out <= kNarrowMost) {
    const int64_t blocks = (p->rows + kNarrowRows - 1) / kNarrowRows, steps = (p->in + kNarrowK - 1) / kNarrowK;
    const double each = (p->out <= 8 ? 0.55 : p->out <= 16 ? 0.75 : 1.1) * (copies_whole(p) ? 1.0 : 1.35);
    if (3.0 + each * static_cast<double>(steps * ((blocks + h->sms - 1) / h->sms)) < std::min(few, tensor))
      return Way::kNarrow;
  }
  return p->rows <= kFewRows && few < tensor ? Way::kFew : Way::kTensor;
}

}  // namespace

extern "C" int64_t pt_b200_linear_work(const pt_b200_ops *h, const pt_b200_linear_args *p) {
  if (!h || !p || !sizes_ok(p->rows, p->in, p->out) || p->rows == 0) return 0;
  if (way(h, p) != Way::kTensor) return 0;
  return operand_bytes(p->dtype, p->x, p->rows, p->in, p->ldx) +
         operand_bytes(p->dtype, p->w, p->out, p->in, p->ldw);
}

extern "C" int pt_b200_linear(pt_b200_ops *h, void *stream, const pt_b200_linear_args *p) {
  PTB_REQUIRE(h && p, "pt_b200_linear: NULL handle or arguments");
  PTB_REQUIRE(p->dtype >= PT_B200_F32 && p->dtype <= PT_B200_F16, "pt_b200_linear: unknown element type %d",
              p->dtype);
  PTB_REQUIRE(p->act == PT_B200_ACT_NONE || p->act == PT_B200_ACT_LEAKY || p->act == PT_B200_ACT_RELU ||
                  p->act == PT_B200_ACT_GELU || p->act == PT_B200_ACT_SILU,
              "pt_b200_linear: unknown activation %d", p->act);
  PTB_REQUIRE(sizes_ok(p->rows, p->in, p->out), "pt_b200_linear: rows %lld, in %lld, out %lld",
              (long long)p->rows, (long long)p->in, (long long)p->out);
  const int eb = dtype_bytes(p->dtype);
  PTB_REQUIRE(rows_ok(p->x, p->rows, p->in, p->ldx, eb) && rows_ok(p->w, p->out, p->in, p->ldw, eb) &&
                  rows_ok(p->y, p->rows, p->out, p->ldy, eb),
              "pt_b200_linear: x, w and y need an aligned pointer and a row stride of at least their columns");
  PTB_REQUIRE((!p->residual || p->ldr >= p->out) && (!p->pre || p->ldp >= p->out),
              "pt_b200_linear: residual and pre need a row stride of at least out");
  PTB_REQUIRE(element_ok(p->bias, eb) && element_ok(p->residual, eb) && element_ok(p->pre, eb),
              "pt_b200_linear: bias, residual or pre is not aligned to its elements");
  if (p->rows == 0) return 0;
  DeviceScope on(h->device);
  PTB_REQUIRE(on.ok, "pt_b200_linear: device %d cannot be used", h->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const LinearEpi epi{p->bias, p->residual, p->y, p->pre, p->ldr, p->ldy, p->ldp, p->act, p->slope};
  const Way by = way(h, p);
  if (by != Way::kTensor) {
    const FewArgs a{p->x, p->w, p->in, p->out, p->ldx, p->ldw, static_cast<int>(p->rows), 1, epi};
    const bool vec = copies_whole(p);
    if (by == Way::kNarrow)
      return p->out <= 8    ? launch_narrow<1>(a, vec, st)
             : p->out <= 16 ? launch_narrow<2>(a, vec, st)
                            : launch_narrow<4>(a, vec, st);
    return with_dtype(p->dtype, [&](auto *z) -> int {
      using T = std::remove_pointer_t<decltype(z)>;
      return vec ? launch_few<T, true>(h, a, st) : launch_few<T, false>(h, a, st);
    });
  }
  const int64_t need = pt_b200_linear_work(h, p);
  PTB_REQUIRE(need == 0 || (p->work && p->work_bytes >= need && reinterpret_cast<uintptr_t>(p->work) % 256 == 0),
              "pt_b200_linear: %lld bytes of 256-byte aligned workspace are needed, %lld given", (long long)need,
              (long long)p->work_bytes);
  char *work = static_cast<char *>(p->work);
  TcProduct q{};
  PrepJobs jobs{};
  int n = 0;
  q.a = operand(h, p->dtype, p->w, p->out, p->in, p->ldw, &work, &jobs, &n);
  q.b = operand(h, p->dtype, p->x, p->rows, p->in, p->ldx, &work, &jobs, &n);
  q.rows = p->rows;
  q.chans = p->out;
  q.k = p->in;
  q.e = epi;
  if (tc_prep(p->dtype, jobs, n, st)) return -1;
  return tc_products(h, p->dtype, &q, 1, ColumnSums{}, n > 0, st);
}

// The gradient's operand dpre is dy itself where nothing has to be computed or copied for it.
static bool grad_direct(const pt_b200_linear_grad_args *p) {
  return p->act == PT_B200_ACT_NONE && tc_direct(p->dtype, p->dy, p->rows, p->lddy);
}

extern "C" int64_t pt_b200_linear_backward_work(const pt_b200_ops *h, const pt_b200_linear_grad_args *p) {
  if (!h || !p || !sizes_ok(p->rows, p->in, p->out) || p->rows == 0) return 0;
  int64_t need = 0;
  if ((p->dx || p->dw) && !grad_direct(p)) need += tc_plane_bytes(p->dtype, p->rows, p->out);
  if (p->dx) need += operand_bytes(p->dtype, p->w, p->out, p->in, p->ldw);
  if (p->dw) need += operand_bytes(p->dtype, p->x, p->rows, p->in, p->ldx);
  if (p->db) need += static_cast<int64_t>(tc_row_blocks(h, p->rows, p->out)) * p->out * 4;
  return need;
}

extern "C" int pt_b200_linear_backward(pt_b200_ops *h, void *stream, const pt_b200_linear_grad_args *p) {
  PTB_REQUIRE(h && p, "pt_b200_linear_backward: NULL handle or arguments");
  PTB_REQUIRE(p->dtype >= PT_B200_F32 && p->dtype <= PT_B200_F16,
              "pt_b200_linear_backward: unknown element type %d", p->dtype);
  PTB_REQUIRE(p->act == PT_B200_ACT_NONE || p->act == PT_B200_ACT_LEAKY || p->act == PT_B200_ACT_RELU ||
                  p->act == PT_B200_ACT_GELU || p->act == PT_B200_ACT_SILU,
              "pt_b200_linear_backward: unknown activation %d", p->act);
  PTB_REQUIRE(sizes_ok(p->rows, p->in, p->out), "pt_b200_linear_backward: rows %lld, in %lld, out %lld",
              (long long)p->rows, (long long)p->in, (long long)p->out);
  const int eb = dtype_bytes(p->dtype);
  const bool acts = p->act != PT_B200_ACT_NONE;
  PTB_REQUIRE(p->dx || p->dw || p->db, "pt_b200_linear_backward: nothing to compute");
  PTB_REQUIRE(rows_ok(p->dy, p->rows, p->out, p->lddy, eb) &&
                  (!acts || rows_ok(p->pre, p->rows, p->out, p->ldp, eb)),
              "pt_b200_linear_backward: dy (and pre where there is an activation) needs an aligned pointer and a "
              "row stride of at least out");
  PTB_REQUIRE((!p->dx || (rows_ok(p->w, p->out, p->in, p->ldw, eb) && p->lddx >= p->in)) &&
                  (!p->dw || (rows_ok(p->x, p->rows, p->in, p->ldx, eb) && p->lddw >= p->in)),
              "pt_b200_linear_backward: dx needs w and dw needs x, with row strides of at least in");
  PTB_REQUIRE(element_ok(p->dx, eb) && element_ok(p->dw, eb) && element_ok(p->db, eb),
              "pt_b200_linear_backward: dx, dw or db is not aligned to its elements");
  DeviceScope on(h->device);
  PTB_REQUIRE(on.ok, "pt_b200_linear_backward: device %d cannot be used", h->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->rows == 0) {   // sums over no rows
    if (p->dw) PTB_CUDA(cudaMemset2DAsync(p->dw, p->lddw * eb, 0, p->in * eb, p->out, st));
    if (p->db) PTB_CUDA(cudaMemsetAsync(p->db, 0, p->out * eb, st));
    return 0;
  }
  const int64_t need = pt_b200_linear_backward_work(h, p);
  PTB_REQUIRE(need == 0 || (p->work && p->work_bytes >= need && reinterpret_cast<uintptr_t>(p->work) % 256 == 0),
              "pt_b200_linear_backward: %lld bytes of 256-byte aligned workspace are needed, %lld given",
              (long long)need, (long long)p->work_bytes);
  char *work = static_cast<char *>(p->work);
  PrepJobs jobs{};
  int n = 0;
  // dpre, its column sums, and the other operands: one pass
  TcOperand g = tc_tensor(p->dy, p->rows, p->out, p->lddy);
  PrepJob j{};
  j.src = p->dy;
  j.pre = p->pre;
  j.rows = p->rows;
  j.cols = p->out;
  j.ld = p->lddy;
  j.ldp = p->ldp;
  j.act = p->act;
  j.slope = p->slope;
  if ((p->dx || p->dw) && !grad_direct(p)) {
    g = tc_planes(work, p->rows, p->out);
    j.dst = work;
    j.ldd = g.ld;
    j.plane = g.plane;
    work += tc_plane_bytes(p->dtype, p->rows, p->out);
  }
  TcProduct products[2] = {};
  int count = 0;
  if (p->dx) {
    TcProduct &dx = products[count++];
    dx.a = operand(h, p->dtype, p->w, p->out, p->in, p->ldw, &work, &jobs, &n);
    dx.b = g;
    dx.a_mn = true;
    dx.rows = p->rows;
    dx.chans = p->in;
    dx.k = p->out;
    dx.e.y = p->dx;
    dx.e.ldy = p->lddx;
  }
  if (p->dw) {
    TcProduct &dw = products[count++];
    dw.a = operand(h, p->dtype, p->x, p->rows, p->in, p->ldx, &work, &jobs, &n);
    dw.b = g;
    dw.a_mn = dw.b_mn = true;
    dw.rows = p->out;
    dw.chans = p->in;
    dw.k = p->rows;
    dw.e.y = p->dw;
    dw.e.ldy = p->lddw;
  }
  ColumnSums sums{};
  if (p->db) {
    j.part = reinterpret_cast<float *>(work);
    sums = ColumnSums{j.part, p->db, tc_row_blocks(h, p->rows, p->out), p->out};
  }
  if (j.dst || j.part) tc_add_job(h, p->dtype, &jobs, &n, j);
  if (tc_prep(p->dtype, jobs, n, st)) return -1;
  if (count) return tc_products(h, p->dtype, products, count, sums, n > 0, st);
  return with_dtype(p->dtype, [&](auto *z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    return reduce_columns<T>(sums.part, sums.parts, sums.n, static_cast<T *>(sums.out), st);
  });
}
