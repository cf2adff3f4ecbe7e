// linear.cuh -- the linear layer's kernels as its host code (linear.cu) calls them.
#pragma once
#include "ops.cuh"

namespace ptb {

// What a product's result goes through on its way out.  Element (m, n) of the product is one
// output element; y, residual and pre are row-major in (m, n).
struct LinearEpi {
  const void *bias;        // [n] or null
  const void *residual;    // [m][n], row stride ldr, or null
  void *y;
  void *pre;               // the value before the activation, or null
  int64_t ldr, ldy, ldp;
  int act;
  float slope;
};

struct ActOnOne {
  float &v;
  float slope;
  template <int ACT>
  __device__ __forceinline__ void operator()() const { v = act_value<ACT>(both(v), slope).x; }
};
template <class T>
__device__ __forceinline__ void linear_store(const LinearEpi &e, int64_t m, int64_t n, float v) {
  if (e.bias) v += to_f32(static_cast<const T *>(e.bias)[n]);
  if (e.pre) static_cast<T *>(e.pre)[m * e.ldp + n] = from_f32<T>(v);
  with_act(e.act, ActOnOne{v, e.slope});
  if (e.residual) v += to_f32(static_cast<const T *>(e.residual)[m * e.ldr + n]);
  static_cast<T *>(e.y)[m * e.ldy + n] = from_f32<T>(v);
}

}  // namespace ptb
