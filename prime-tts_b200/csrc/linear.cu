// linear.cu -- pt_b200_linear and its gradient.
//
//   pre = x W^T + b;  y = act(pre) + r
//   dpre = dy * act'(pre);  dx = dpre W;  dW = dpre^T x;  db = sum over rows of dpre
//
// The three products run on the tensor cores (linear_tc.cu).
#include "linear_tc.cuh"

using namespace ptb;

namespace {

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

}  // namespace

extern "C" int64_t pt_b200_linear_work(const pt_b200_ops *h, const pt_b200_linear_args *p) {
  if (!h || !p || !sizes_ok(p->rows, p->in, p->out) || p->rows == 0) return 0;
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
  q.e = LinearEpi{p->bias, p->residual, p->y, p->pre, p->ldr, p->ldy, p->ldp, p->act, p->slope};
  if (tc_prep(p->dtype, jobs, n, st)) return -1;
  return tc_product(h, p->dtype, q, ColumnSums{}, n > 0, false, st);
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
  TcProduct dx{}, dw{};
  if (p->dx) dx.a = operand(h, p->dtype, p->w, p->out, p->in, p->ldw, &work, &jobs, &n);
  if (p->dw) dw.a = operand(h, p->dtype, p->x, p->rows, p->in, p->ldx, &work, &jobs, &n);
  ColumnSums sums{};
  if (p->db) {
    j.part = reinterpret_cast<float *>(work);
    sums = ColumnSums{j.part, p->db, tc_row_blocks(h, p->rows, p->out), p->out};
  }
  if (j.dst || j.part) tc_add_job(h, p->dtype, &jobs, &n, j);
  if (tc_prep(p->dtype, jobs, n, st)) return -1;
  if (p->dx) {
    dx.b = g;
    dx.a_mn = true;
    dx.rows = p->rows;
    dx.chans = p->in;
    dx.k = p->out;
    dx.e.y = p->dx;
    dx.e.ldy = p->lddx;
    if (tc_product(h, p->dtype, dx, sums, n > 0, false, st)) return -1;
    sums = ColumnSums{};
  }
  if (p->dw) {
    dw.b = g;
    dw.a_mn = dw.b_mn = true;
    dw.rows = p->out;
    dw.chans = p->in;
    dw.k = p->rows;
    dw.e.y = p->dw;
    dw.e.ldy = p->lddw;
    // dx and dW need the same passes and nothing of each other
    if (tc_product(h, p->dtype, dw, sums, n > 0 || p->dx, p->dx != nullptr, st)) return -1;
    sums = ColumnSums{};
  }
  if (sums.parts == 0) return 0;
  return with_dtype(p->dtype, [&](auto *z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    return reduce_columns<T>(sums.part, sums.parts, sums.n, static_cast<T *>(sums.out), st);
  });
}
