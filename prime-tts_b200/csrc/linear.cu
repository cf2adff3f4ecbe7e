// linear.cu -- pt_b200_linear and its gradient.
//
//   pre = x W^T + b;  y = act(pre) + r
//   dpre = dy * act'(pre);  dx = dpre W;  dW = dpre^T x;  db = sum over rows of dpre
//
// The three products run on the tensor cores (linear_tc.cu).
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

// Whether a call takes the few-rows kernel: by the microseconds that both would take.  Its own follow
// from its warps' tasks (two channels x eight rows), each a start and k; the tensor cores' from a start,
// the first stages of k, the weights and x (in its planes, against a tile of 128 channels).  Fits to measurements (the tensor cores' in brackets, rows x
// in x out):
//   bf16  4 x 4096 x 1024 4.5 (6.8), 8 x 1024 x 1024 3.9 (5.9), 2 x 4096 x 4096 7.4 (8.8), 4 x 4096 x
//         4096 10.5 (8.8), 64 x 192 x 768 5.7 (4.9), 1000 x 64 x 64 6.2 (4.5)
//   not aligned, so that the tensor cores need copies: 128 x 101 x 201 4.4 (5.9), 500 x 101 x 201 10.1
//         (5.9), 4 x 4001 x 4001 16.3 (21), 8 x 4001 x 4001 25.6 (21)
//   fp32, which the tensor cores need in planes: 8 x 4096 x 4096 15.6 (48), 16 x 192 x 768 3.2 (8.7),
//         128 x 768 x 192 5.3 (9.9), 2000 x 192 x 16 3.3 (9.4), 700 x 192 x 192 7.4 (9.1), 7369 x
//         2296 x 24 46 (68), 16064 x 347 x 40 (27)
constexpr int kFewRows = 1 << 18;
bool few_rows(const pt_b200_linear_args *p) {
  if (p->rows > kFewRows) return false;
  const bool f32 = p->dtype == PT_B200_F32;
  const bool direct = tc_direct(p->dtype, p->x, p->rows, p->ldx) && tc_direct(p->dtype, p->w, p->out, p->ldw);
  const double k = static_cast<double>(p->in), w = k * static_cast<double>(p->out) * 1e-6;
  const double tasks = static_cast<double>((p->rows + kFewGroup - 1) / kFewGroup) * ((p->out + 1) / 2) * 1e-3;
  const double fill = p->rows <= 1 ? 0.125 : p->rows <= 2 ? 0.25 : p->rows <= 4 ? 0.5 : 1.0;   // rows a task has
  const double four = p->rows > 4 && tasks > 2.4 ? 0.7 : 1.0;   // many tasks, of four channels each
  const double few = 2.4 + four * tasks * (0.7 + fill * k * (f32 ? 0.0014 : direct ? 0.0018 : 0.003));
  const double start = 0.001 * (k < 1024 ? k : 1024), x = static_cast<double>(p->rows) * k * 1e-6;
  return few < start + (f32 ? 7.6 + 2.4 * w + 4.0 * x : direct ? 4.6 + 0.18 * w + 0.6 * x : 5.7 + 0.9 * w + 1.4 * x);
}

}  // namespace

extern "C" int64_t pt_b200_linear_work(const pt_b200_ops *h, const pt_b200_linear_args *p) {
  if (!h || !p || !sizes_ok(p->rows, p->in, p->out) || p->rows == 0) return 0;
  if (few_rows(p)) return 0;
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
              "pt_b200_linear: x, w and y need a pointer and a row stride of at least their columns");
  PTB_REQUIRE((!p->residual || p->ldr >= p->out) && (!p->pre || p->ldp >= p->out),
              "pt_b200_linear: residual and pre need a row stride of at least out");
  if (p->rows == 0) return 0;
  DeviceScope on(h->device);
  PTB_REQUIRE(on.ok, "pt_b200_linear: device %d cannot be used", h->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const LinearEpi epi{p->bias, p->residual, p->y, p->pre, p->ldr, p->ldy, p->ldp, p->act, p->slope};
  if (few_rows(p)) {
    const FewArgs a{p->x, p->w, p->in, p->out, p->ldx, p->ldw, static_cast<int>(p->rows), 1, epi};
    const int v = 16 / eb;
    auto aligned = [&](const void *q, int64_t rows, int64_t ld) {
      return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (rows == 1 || ld % v == 0);
    };
    const bool vec = p->in % v == 0 && aligned(p->x, p->rows, p->ldx) && aligned(p->w, p->out, p->ldw);
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
              "pt_b200_linear_backward: dy (and pre where there is an activation) needs a pointer and a "
              "row stride of at least out");
  PTB_REQUIRE((!p->dx || (rows_ok(p->w, p->out, p->in, p->ldw, eb) && p->lddx >= p->in)) &&
                  (!p->dw || (rows_ok(p->x, p->rows, p->in, p->ldx, eb) && p->lddw >= p->in)),
              "pt_b200_linear_backward: dx needs w and dw needs x, with row strides of at least in");
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
