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

// fp32 as three bf16 values, x = o0 + 2^-7 o1 + 2^-14 o2: each is under 2^-8 of the one before (2^-7
// where that was truncated), so the scaled ones stay below x and reach bf16's smallest numbers no sooner
// than x itself.  A value that is not finite lies in the first alone; one that would round up to infinity
// is truncated there instead.
constexpr int kPlaneShift = 7;
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&o)[3]) {
  constexpr float kUp = 1 << kPlaneShift;
  o[0] = __float2bfloat16_rn(x);
  if (!(fabsf(x) <= 3.38953139e38f)) {   // beyond the largest finite bf16, or NaN
    if (!isfinite(x)) {
      o[1] = o[2] = __float2bfloat16_rn(0.0f);
      return;
    }
    o[0] = __float2bfloat16_rz(x);
  }
  const float r1 = (x - __bfloat162float(o[0])) * kUp;
  o[1] = __float2bfloat16_rn(r1);
  o[2] = __float2bfloat16_rn((r1 - __bfloat162float(o[1])) * kUp);
}

// One pass over a matrix that makes an operand of it: dst receives src * act'(pre) (src itself
// without an activation) in the rows and planes the tensor cores read, part its column sums, one
// row of partials per block of rows.  dst or part may be null.
struct PrepJob {
  const void *src, *pre;
  void *dst;
  float *part;
  int64_t rows, cols, ld, ldp, ldd, plane;
  int act;
  float slope;
  int lanes;                   // threads across the columns, 8 columns each (a power of two)
  int col_blocks, row_blocks;
  bool vec;
};
constexpr int kMaxJobs = 3;
struct PrepJobs {
  PrepJob j[kMaxJobs];
  int end[kMaxJobs];           // running count of blocks
};

// Once per handle: the kernels' shared memory, and how many of their clusters fit the GPU.
int tc_setup(pt_b200_ops *h);
// Whether a tensor can be read where it lies; else the bytes of its planes.
bool tc_direct(int dtype, const void *p, int64_t rows, int64_t ld);
int64_t tc_plane_bytes(int dtype, int64_t rows, int64_t cols);
TcOperand tc_tensor(const void *p, int64_t rows, int64_t cols, int64_t ld);
TcOperand tc_planes(void *p, int64_t rows, int64_t cols);
// Adds a pass to `jobs` (one launch runs them all) and gives the rows of partials it will write.
int tc_row_blocks(const pt_b200_ops *h, int64_t rows, int64_t cols);
void tc_add_job(const pt_b200_ops *h, int dtype, PrepJobs *jobs, int *n, PrepJob job);
int tc_prep(int dtype, const PrepJobs &jobs, int n, cudaStream_t st);
// One product, or two that need nothing of each other.  After a kernel of the same call that lets
// them start early, `early` hides the launch behind it; `sums` is work that epilogue warps do while
// the first tile's products run.
int tc_products(const pt_b200_ops *h, int dtype, const TcProduct *p, int count, const ColumnSums &sums, bool early,
                cudaStream_t st);

}  // namespace ptb
