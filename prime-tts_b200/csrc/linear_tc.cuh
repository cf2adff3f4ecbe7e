// linear_tc.cuh -- the tensor-core products of the linear layer (linear_tc.cu).
#pragma once
#include "linear.cuh"

namespace ptb {

// A matrix the tensor cores can read: 2-byte elements, row-major, 16-byte aligned rows; `plane`
// elements from one of the three planes of an fp32 matrix to the next.
struct TcOperand {
  const void *p;
  int64_t rows, cols, ld, plane;
};

// D[row][chan] = sum_k A(chan, k) B(row, k).  An operand's rows are its product index and its
// columns k, or (mn) the other way round.
struct TcProduct {
  TcOperand a, b;
  bool a_mn, b_mn;
  int64_t rows, chans, k;
  LinearEpi e;
};

// fp32 as the sum of three bf16 values.  One that is not finite lies in the first alone; one that
// would round up to infinity is truncated there instead.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&o)[3]) {
  o[0] = __float2bfloat16_rn(x);
  if (!isfinite(__bfloat162float(o[0]))) {
    if (!isfinite(x)) {
      o[1] = o[2] = __float2bfloat16_rn(0.0f);
      return;
    }
    o[0] = __float2bfloat16_rz(x);
  }
  const float r1 = x - __bfloat162float(o[0]);
  o[1] = __float2bfloat16_rn(r1);
  o[2] = __float2bfloat16_rn(r1 - __bfloat162float(o[1]));
}

struct PackArgs {
  const void *src;
  void *dst;
  int64_t rows, cols, ld, ld_out, plane;
};

// Whether a tensor can be read where it lies; else the bytes of its planes.
bool tc_direct(int dtype, const void *p, int64_t rows, int64_t ld);
int64_t tc_plane_bytes(int dtype, int64_t rows, int64_t cols);
TcOperand tc_tensor(const void *p, int64_t rows, int64_t cols, int64_t ld);
TcOperand tc_planes(void *p, int64_t rows, int64_t cols);
int tc_pack(const pt_b200_ops *h, int dtype, const void *src, int64_t ld, const TcOperand &to, cudaStream_t st);
int tc_product(const pt_b200_ops *h, int dtype, const TcProduct &p, cudaStream_t st);

}  // namespace ptb
