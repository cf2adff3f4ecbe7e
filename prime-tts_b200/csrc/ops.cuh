// ops.cuh -- shared by the transformer-layer operators (linear.cu, layernorm.cu, ops.cu): element
// types, activations, the handle, and the launch checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/pt_b200.h"
#include "common.cuh"

struct pt_b200_ops {
  int device;
  int sms;
  uint32_t *gerr;    // device error word: bounded waits that gave up
  int clusters[4];   // tensor-core kernels: clusters of 1, 2, 4, 8 blocks that run at once
};

namespace ptb {

// Makes the handle's device current for one call and puts the caller's back afterwards.
struct DeviceScope {
  int prev = -1;
  bool ok = false;
  explicit DeviceScope(int device) {
    int cur = -1;
    if (cudaGetDevice(&cur) != cudaSuccess) return;
    if (cur != device) {
      if (cudaSetDevice(device) != cudaSuccess) return;
      prev = cur;
    }
    ok = true;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// ---- element types: every sum, statistic and activation is computed in fp32; a value is rounded
// to the tensor's type (to nearest even) only when it is stored.
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements moved as one access (V * sizeof(T) = 16 bytes, or one element).
template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// Runs fn with a null pointer of the C type that `dtype` names.
template <class F>
int with_dtype(int dtype, F &&fn) {
  switch (dtype) {
    case PT_B200_F32: return fn(static_cast<float *>(nullptr));
    case PT_B200_BF16: return fn(static_cast<__nv_bfloat16 *>(nullptr));
    case PT_B200_F16: return fn(static_cast<__half *>(nullptr));
  }
  set_error("pt_b200: unknown element type %d", dtype);
  return -1;
}
inline int dtype_bytes(int dtype) { return dtype == PT_B200_F32 ? 4 : 2; }

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// ---- activations.  A NaN passes through each of them; the slope of relu and leaky at 0 is that
// of the side the comparison puts it on (relu 0, leaky 1).
//
// The normal distribution function is h(-p) below 0 and 1 - h(p) from there on, with h(p) = erfc(p / sqrt 2)
// / 2 = exp(-p^2 / 2) t Q(t), t = 1 / (1 + 0.3 p).  Q has degree 7 and Q(1) = 1/2; its coefficients are
// those of the least largest error on 0 <= p <= 14.5 in the weight h^(1/2) (Lawson's iteration of weighted
// least squares): 1.0e-8 of h in all, and 1.1e-6 relative out to h = 1e-47, so that gelu's left tail keeps
// its digits.  (Degree 6 leaves 5.9e-8.  Abramowitz and Stegun's 7.1.26, one term less still, is off by
// 7.5e-8: gelu of normal arguments had an error of 5.7e-8, and has 2.6e-8 now, as an fp32 erf.)  The
// exponential is also the density's, so value and slope of gelu cost one exponential and one reciprocal.
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// The hardware's 2^x and 1 / x (errors of about 2^-22), denormal results as zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ void normal_cdf(float2 p, float2 *cdf, float2 *gauss) {
  const float2 a = mul2(mul2(p, p), both(-0.5f * kLog2E));
  const float2 e = make_float2(exp2_fast(a.x), exp2_fast(a.y));
  const float2 d = fma2(both(0.3f), make_float2(fabsf(p.x), fabsf(p.y)), both(1.0f));
  const float2 t = make_float2(rcp_fast(d.x), rcp_fast(d.y));
  float2 q = fma2(both(0.03523390028f), t, both(-0.1546597141f));
  q = fma2(q, t, both(0.2006010744f));
  q = fma2(q, t, both(-0.04699237243f));
  q = fma2(q, t, both(0.1242275003f));
  q = fma2(q, t, both(0.1014719389f));
  q = fma2(q, t, both(0.120467785f));
  q = mul2(fma2(q, t, both(0.1196498876f)), t);
  const float2 lo = mul2(q, e), hi = fma2(q, make_float2(-e.x, -e.y), both(1.0f));
  *cdf = make_float2(p.x < 0.0f ? lo.x : hi.x, p.y < 0.0f ? lo.y : hi.y);
  *gauss = e;
}

// Value and slope of two arguments at once.
template <int ACT>
__device__ __forceinline__ float2 act_value(float2 p, float slope) {
  if constexpr (ACT == PT_B200_ACT_LEAKY)
    return make_float2(p.x < 0.0f ? slope * p.x : p.x, p.y < 0.0f ? slope * p.y : p.y);
  if constexpr (ACT == PT_B200_ACT_RELU) return make_float2(p.x < 0.0f ? 0.0f : p.x, p.y < 0.0f ? 0.0f : p.y);
  if constexpr (ACT == PT_B200_ACT_GELU) {
    float2 cdf, gauss;
    normal_cdf(p, &cdf, &gauss);
    return mul2(p, cdf);
  }
  if constexpr (ACT == PT_B200_ACT_SILU) {
    const float2 a = mul2(p, both(-kLog2E));
    return mul2(p, make_float2(rcp_fast(1.0f + exp2_fast(a.x)), rcp_fast(1.0f + exp2_fast(a.y))));
  }
  return p;
}

template <int ACT>
__device__ __forceinline__ float2 act_grad(float2 p, float slope) {
  if constexpr (ACT == PT_B200_ACT_LEAKY) return make_float2(p.x < 0.0f ? slope : 1.0f, p.y < 0.0f ? slope : 1.0f);
  if constexpr (ACT == PT_B200_ACT_RELU) return make_float2(p.x <= 0.0f ? 0.0f : 1.0f, p.y <= 0.0f ? 0.0f : 1.0f);
  if constexpr (ACT == PT_B200_ACT_GELU) {
    float2 cdf, gauss;
    normal_cdf(p, &cdf, &gauss);
    return fma2(mul2(p, both(kInvSqrt2Pi)), gauss, cdf);
  }
  if constexpr (ACT == PT_B200_ACT_SILU) {
    const float2 a = mul2(p, both(-kLog2E));
    const float2 s = make_float2(rcp_fast(1.0f + exp2_fast(a.x)), rcp_fast(1.0f + exp2_fast(a.y)));
    // s (1 + p (1 - s))
    return fma2(mul2(s, p), add2(both(1.0f), make_float2(-s.x, -s.y)), s);
  }
  return both(1.0f);
}

// fn.template operator()<ACT>() for the activation's code: the choice is made once, outside loops.
template <class F>
__device__ __forceinline__ void with_act(int act, F &&fn) {
  switch (act) {
    case PT_B200_ACT_LEAKY: fn.template operator()<PT_B200_ACT_LEAKY>(); break;
    case PT_B200_ACT_RELU: fn.template operator()<PT_B200_ACT_RELU>(); break;
    case PT_B200_ACT_GELU: fn.template operator()<PT_B200_ACT_GELU>(); break;
    case PT_B200_ACT_SILU: fn.template operator()<PT_B200_ACT_SILU>(); break;
    default: fn.template operator()<PT_B200_ACT_NONE>();
  }
}

// Lets the next kernel of the stream start before this one ends (it waits below for its results).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Waits for the kernels before this one, where it was launched to start early; else does nothing.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Columns of partial sums [parts][n] -> T out[n] (layernorm.cu).  A column's partials are added by
// eight lanes, each every eighth of them, and the lanes' sums in order.
struct ColumnSums {
  const float *part;
  void *out;
  int parts;
  int64_t n;
};
// One lane's partials p, p + step, ... below parts: four sums in turns, which are shorter than one (db of 3616
// rows of 192 fp32 had an error of 1.53e-7 with one), added in pairs.
__device__ __forceinline__ float lane_sum(const float *column, int p, int parts, int step, int64_t n) {
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (; p + 7 * step < parts; p += 8 * step)   // (eight loads in flight)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i % 4] += column[(p + i * step) * n];
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (p + i * step < parts) v[i % 4] += column[(p + i * step) * n];
  return (v[0] + v[1]) + (v[2] + v[3]);
}
template <class T>
int reduce_columns(const float *part, int parts, int64_t n, T *out, cudaStream_t st);

// ---- argument checks shared by the entry points: a kernel reads and writes whole elements, so a
// pointer that is not aligned to its element would be an address fault on the device
inline bool element_ok(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }
inline bool rows_ok(const void *p, int64_t rows, int64_t cols, int64_t ld, int bytes) {
  return rows == 0 || (p && ld >= cols && element_ok(p, bytes));
}

}  // namespace ptb
