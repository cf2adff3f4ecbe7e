// linear.cu -- pt_b200_linear and its gradient.
//
//   pre = x W^T + b;  y = act(pre) + r
//   dpre = dy * act'(pre);  dx = dpre W;  dW = dpre^T x;  db = sum over rows of dpre
//
// All three products are D[m][n] = sum_k A(m, k) B(n, k) over operands read along either index.
#include "linear.cuh"

using namespace ptb;

namespace {

constexpr int kBlock = 256;

// ---- fp32 FMA product for every type, stride and size: 64 x 64 outputs per block, 4 x 4 per
// thread, operands staged 16 deep in shared memory as fp32.
constexpr int kTile = 64, kDepth = 16;

template <class T>
__global__ void __launch_bounds__(kBlock) product_kernel(const LinearProduct p) {
  __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
  const int64_t tn = (p.n + kTile - 1) / kTile;
  const int64_t m0 = blockIdx.x / tn * kTile, n0 = blockIdx.x % tn * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const T *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b);
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kDepth) {
#pragma unroll
    for (int i = 0; i < kTile * kDepth / kBlock; ++i) {
      const int e = i * kBlock + threadIdx.x;
      // consecutive threads follow the index that is contiguous in memory
      const int ka = p.a_k == 1 ? e % kDepth : e / kTile, ra = p.a_k == 1 ? e / kDepth : e % kTile;
      const int kb = p.b_k == 1 ? e % kDepth : e / kTile, rb = p.b_k == 1 ? e / kDepth : e % kTile;
      sa[ka][ra] = m0 + ra < p.m && k0 + ka < p.k
                       ? to_f32(a[(m0 + ra) * p.a_m + (k0 + ka) * p.a_k]) : 0.0f;
      sb[kb][rb] = n0 + rb < p.n && k0 + kb < p.k
                       ? to_f32(b[(n0 + rb) * p.b_n + (k0 + kb) * p.b_k]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      float va[4], vb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        va[i] = sa[k][ty * 4 + i];
        vb[i] = sb[k][tx + 16 * i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(va[i], vb[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (m0 + ty * 4 + i < p.m && n0 + tx + 16 * j < p.n)
        linear_store<T>(p.e, m0 + ty * 4 + i, n0 + tx + 16 * j, acc[i][j]);
}

template <class T>
int launch_product(const LinearProduct &p, cudaStream_t st) {
  const int64_t tiles = ((p.m + kTile - 1) / kTile) * ((p.n + kTile - 1) / kTile);
  PTB_REQUIRE(tiles < (int64_t(1) << 31), "pt_b200: product of %lld x %lld is too large", (long long)p.m,
              (long long)p.n);
  product_kernel<T><<<static_cast<unsigned>(tiles), kBlock, 0, st>>>(p);
  PTB_CUDA(cudaGetLastError());
  count_launch();
  return 0;
}

// ---- dpre = dy * act'(pre), and its column sums as one row of partials per blockIdx.y
struct GradArgs {
  const void *dy, *pre;
  void *g;               // dpre, or null (no activation: dpre is dy itself)
  float *part;           // [gridDim.y][n], or null
  int64_t rows, n, lddy, ldp, ldg;
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
      if (a.act) d *= act_grad(to_f32(static_cast<const T *>(a.pre)[r * a.ldp + c]), a.act, a.slope);
      // rounded to the operands' type for the two products; the sums take the fp32 value
      if (a.g) static_cast<T *>(a.g)[r * a.ldg + c] = from_f32<T>(d);
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

int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

bool sizes_ok(int64_t rows, int64_t n_in, int64_t n_out) {
  return rows >= 0 && n_in > 0 && n_out > 0 && rows < (int64_t(1) << 31) && n_in < (int64_t(1) << 30) &&
         n_out < (int64_t(1) << 30);
}

}  // namespace

extern "C" int64_t pt_b200_linear_work(const pt_b200_ops *h, const pt_b200_linear_args *p) {
  (void)h;
  (void)p;
  return 0;
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
  LinearProduct q{p->x, p->w, p->ldx, 1, p->ldw, 1, p->rows, p->out, p->in,
                  {p->bias, p->residual, p->y, p->pre, p->ldr, p->ldy, p->ldp, p->act, p->slope}};
  return with_dtype(p->dtype, [&](auto *z) -> int {
    return launch_product<std::remove_pointer_t<decltype(z)>>(q, st);
  });
}

extern "C" int64_t pt_b200_linear_backward_work(const pt_b200_ops *h, const pt_b200_linear_grad_args *p) {
  if (!h || !p || !sizes_ok(p->rows, p->in, p->out) || p->rows == 0) return 0;
  int64_t need = 0;
  if (p->act != PT_B200_ACT_NONE) need += up256(p->rows * p->out * dtype_bytes(p->dtype));
  if (p->db) need += up256(static_cast<int64_t>(grad_parts(p->rows)) * p->out * 4);
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
  PTB_REQUIRE(need == 0 || (p->work && p->work_bytes >= need && reinterpret_cast<uintptr_t>(p->work) % 16 == 0),
              "pt_b200_linear_backward: %lld bytes of 16-byte aligned workspace are needed, %lld given",
              (long long)need, (long long)p->work_bytes);
  return with_dtype(p->dtype, [&](auto *z) -> int {
    using T = std::remove_pointer_t<decltype(z)>;
    char *work = static_cast<char *>(p->work);
    const void *g = p->dy;
    int64_t ldg = p->lddy;
    GradArgs ga{p->dy, p->pre, nullptr, nullptr, p->rows, p->out, p->lddy, p->ldp, p->out, p->act, p->slope};
    if (acts) {
      ga.g = work;
      g = work;
      ldg = p->out;
      work += up256(p->rows * p->out * eb);
    }
    if (p->db) ga.part = reinterpret_cast<float *>(work);
    if (ga.g || ga.part) {
      const int parts = grad_parts(p->rows);
      act_grad_kernel<T><<<dim3(static_cast<unsigned>((p->out + 31) / 32), parts), kBlock, 0, st>>>(ga);
      PTB_CUDA(cudaGetLastError());
      count_launch();
      if (p->db && reduce_columns<T>(ga.part, parts, p->out, static_cast<T *>(p->db), st)) return -1;
    }
    LinearEpi plain{};
    if (p->dx) {
      LinearProduct q{g, p->w, ldg, 1, 1, p->ldw, p->rows, p->in, p->out, plain};
      q.e.y = p->dx;
      q.e.ldy = p->lddx;
      if (launch_product<T>(q, st)) return -1;
    }
    if (p->dw) {
      LinearProduct q{g, p->x, 1, ldg, 1, p->ldx, p->out, p->in, p->rows, plain};
      q.e.y = p->dw;
      q.e.ldy = p->lddw;
      if (launch_product<T>(q, st)) return -1;
    }
    return 0;
  });
}
