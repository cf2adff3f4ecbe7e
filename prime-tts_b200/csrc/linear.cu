// linear.cu -- pt_b200_linear and its gradient.
//
//   pre = x W^T + b;  y = act(pre) + r
//   dpre = dy * act'(pre);  dx = dpre W;  dW = dpre^T x;  db = sum over rows of dpre
//
// The three products run on the tensor cores (linear_tc.cu).
#include "linear_tc.cuh"

using namespace ptb;

namespace {

constexpr int kBlock = 256;

// ---- dpre = dy * act'(pre), and its column sums as one row of partials per blockIdx.y
struct GradArgs {
  const void *dy, *pre;
  void *g;               // dpre as the products read it, or null
  float *part;           // [gridDim.y][n], or null
  int64_t rows, n, lddy, ldp, ldg, plane;
  int act;
  float slope;
};

template <class T>
__global__ void __launch_bounds__(kBlock) act_grad_kernel(const GradArgs a) {
  __shared__ float s[8][33];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int lane = threadIdx.x >> 5;
  float sum = 0.0f;
  if (c < a.n)
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + lane; r < a.rows;
         r += static_cast<int64_t>(gridDim.y) * 8) {
      float d = to_f32(static_cast<const T *>(a.dy)[r * a.lddy + c]);
      // (an explicit product: the sum must not depend on whether d is also stored)
      if (a.act)
        d = __fmul_rn(d, act_grad(to_f32(static_cast<const T *>(a.pre)[r * a.ldp + c]), a.act, a.slope));
      // rounded to the operands' type for the two products; the sums take the fp32 value
      if (a.g) {
        if constexpr (sizeof(T) == 4) {
          __nv_bfloat16 o[3];
          split3(d, o);
#pragma unroll
          for (int p = 0; p < 3; ++p)
            static_cast<__nv_bfloat16 *>(a.g)[p * a.plane + r * a.ldg + c] = o[p];
        } else {
          static_cast<T *>(a.g)[r * a.ldg + c] = from_f32<T>(d);
        }
      }
      sum += d;
    }
  if (!a.part) return;
  s[lane][threadIdx.x & 31] = sum;
  __syncthreads();
  if (threadIdx.x < 32 && c < a.n) {
    sum = 0.0f;
    for (int i = 0; i < 8; ++i) sum += s[i][threadIdx.x];
    a.part[static_cast<int64_t>(blockIdx.y) * a.n + c] = sum;
  }
}

int grad_parts(int64_t rows) {
  const int64_t n = (rows + 63) / 64;
  return static_cast<int>(n < 64 ? n : 64);
}

// An operand: the tensor itself where the tensor cores can read it, else its planes at *work.
struct Operand {
  bool direct;
  int64_t bytes;
};
Operand operand(int dtype, const void *p, int64_t rows, int64_t cols, int64_t ld) {
  const bool direct = tc_direct(dtype, p, rows, ld);
  return Operand{direct, direct ? 0 : tc_plane_bytes(dtype, rows, cols)};
}
int prepare(const pt_b200_ops *h, int dtype, const void *p, int64_t rows, int64_t cols, int64_t ld, char **work,
            TcOperand *out, cudaStream_t st) {
  const Operand o = operand(dtype, p, rows, cols, ld);
  if (o.direct) {
    *out = tc_tensor(p, rows, cols, ld);
    return 0;
  }
  *out = tc_planes(*work, rows, cols);
  *work += o.bytes;
  return tc_pack(h, dtype, p, ld, *out, st);
}

bool sizes_ok(int64_t rows, int64_t n_in, int64_t n_out) {
  return rows >= 0 && n_in > 0 && n_out > 0 && rows < (int64_t(1) << 31) && n_in < (int64_t(1) << 30) &&
         n_out < (int64_t(1) << 30);
}

}  // namespace

extern "C" int64_t pt_b200_linear_work(const pt_b200_ops *h, const pt_b200_linear_args *p) {
  if (!h || !p || !sizes_ok(p->rows, p->in, p->out) || p->rows == 0) return 0;
  return operand(p->dtype, p->x, p->rows, p->in, p->ldx).bytes +
         operand(p->dtype, p->w, p->out, p->in, p->ldw).bytes;
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
  const int64_t need = pt_b200_linear_work(h, p);
  PTB_REQUIRE(need == 0 || (p->work && p->work_bytes >= need && reinterpret_cast<uintptr_t>(p->work) % 256 == 0),
              "pt_b200_linear: %lld bytes of 256-byte aligned workspace are needed, %lld given", (long long)need,
              (long long)p->work_bytes);
  char *work = static_cast<char *>(p->work);
  TcProduct q{};
  if (prepare(h, p->dtype, p->w, p->out, p->in, p->ldw, &work, &q.a, st) ||
      prepare(h, p->dtype, p->x, p->rows, p->in, p->ldx, &work, &q.b, st))
    return -1;
  q.rows = p->rows;
  q.chans = p->out;
  q.k = p->in;
  q.e = LinearEpi{p->bias, p->residual, p->y, p->pre, p->ldr, p->ldy, p->ldp, p->act, p->slope};
  return tc_product(h, p->dtype, q, st);
}

// The gradient's operand dpre is dy itself where nothing has to be computed or copied for it.
static bool grad_direct(const pt_b200_linear_grad_args *p) {
  return p->act == PT_B200_ACT_NONE && tc_direct(p->dtype, p->dy, p->rows, p->lddy);
}

extern "C" int64_t pt_b200_linear_backward_work(const pt_b200_ops *h, const pt_b200_linear_grad_args *p) {
  if (!h || !p || !sizes_ok(p->rows, p->in, p->out) || p->rows == 0) return 0;
  int64_t need = 0;
  if ((p->dx || p->dw) && !grad_direct(p)) need += tc_plane_bytes(p->dtype, p->rows, p->out);
  if (p->dx) need += operand(p->dtype, p->w, p->out, p->in, p->ldw).bytes;
  if (p->dw) need += operand(p->dtype, p->x, p->rows, p->in, p->ldx).bytes;
  if (p->db) need += static_cast<int64_t>(grad_parts(p->rows)) * p->out * 4;
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
  return with_dtype(p->dtype, [&](auto *z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    char *work = static_cast<char *>(p->work);
    TcOperand g = tc_tensor(p->dy, p->rows, p->out, p->lddy);
    GradArgs ga{p->dy, p->pre, nullptr, nullptr, p->rows, p->out, p->lddy, p->ldp, 0, 0, p->act, p->slope};
    if ((p->dx || p->dw) && !grad_direct(p)) {
      g = tc_planes(work, p->rows, p->out);
      ga.g = work;
      ga.ldg = g.ld;
      ga.plane = g.plane;
      work += tc_plane_bytes(p->dtype, p->rows, p->out);
    }
    TcProduct dx{}, dw{};
    if ((p->dx && prepare(h, p->dtype, p->w, p->out, p->in, p->ldw, &work, &dx.a, st)) ||
        (p->dw && prepare(h, p->dtype, p->x, p->rows, p->in, p->ldx, &work, &dw.a, st)))
      return -1;
    if (p->db) ga.part = reinterpret_cast<float *>(work);
    if (ga.g || ga.part) {
      const int parts = grad_parts(p->rows);
      act_grad_kernel<T><<<dim3(static_cast<unsigned>((p->out + 31) / 32), parts), kBlock, 0, st>>>(ga);
      PTB_CUDA(cudaGetLastError());
      count_launch();
      if (p->db && reduce_columns<T>(ga.part, parts, p->out, static_cast<T *>(p->db), st)) return -1;
    }
    if (p->dx) {
      dx.b = g;
      dx.a_mn = true;
      dx.rows = p->rows;
      dx.chans = p->in;
      dx.k = p->out;
      dx.e.y = p->dx;
      dx.e.ldy = p->lddx;
      if (tc_product(h, p->dtype, dx, st)) return -1;
    }
    if (p->dw) {
      dw.b = g;
      dw.a_mn = dw.b_mn = true;
      dw.rows = p->out;
      dw.chans = p->in;
      dw.k = p->rows;
      dw.e.y = p->dw;
      dw.e.ldy = p->lddw;
      if (tc_product(h, p->dtype, dw, st)) return -1;
    }
    return 0;
  });
}
