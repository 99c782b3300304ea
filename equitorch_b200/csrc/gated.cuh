// A gated linear layer, h = act(x W0) * (x W1): what its kernels share.
//
//   x (n, C), W (2, C, F)      a = x W0,  u = x W1,  h = act(a) u
//   backward, from g = dL/dh:  da = g u act'(a),  du = g act(a)          (both projections are formed again, nothing is kept)
//                              dx = da W0^T + du W1^T,   dW0 = x^T da,  dW1 = x^T du
#pragma once

#include "tc_common.cuh"

namespace eqt {
namespace gated {

struct GatedArgs {
  const void *x, *w, *g;
  void *h, *d;               // d (2, n, F): da, du
  void *dx, *dw;
  void* parts;               // (splits, 2, C, F) of the arithmetic type: sums over parts of the rows
  int64_t n;
  int c, f, act;
  int x_pitch, w_pitch, d_pitch;    // values between two rows of x, of W, of da, du and the parts
  int splits;
  int64_t split_rows;
  int* status;
};

// act(a) and its derivative in the arithmetic type
template <typename A> struct Value { A y, dy; };
template <typename A> __device__ __forceinline__ A exp_neg(A x);
template <> __device__ __forceinline__ float exp_neg(float x) {            // results below 2^-126 are zero, which saves their scaling
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * -1.4426950408889634f));
  return y;
}
template <> __device__ __forceinline__ double exp_neg(double x) { return exp(-x); }
template <typename A> __device__ __forceinline__ A inverse(A x);
template <> __device__ __forceinline__ float inverse(float x) {            // one unit in the last place; 0 at infinity
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <> __device__ __forceinline__ double inverse(double x) { return 1.0 / x; }

template <typename A> __device__ __forceinline__ Value<A> activate(A a, int act) {
  if (act == EQT_ACT_RELU) return {a > A(0) || a != a ? a : A(0), a > A(0) ? A(1) : A(0)};
  if (act == EQT_ACT_GELU) {
    const A half = A(0.5) + A(0.5) * (A)erf(a * A(0.70710678118654752));
    return {a * half, half + a * A(0.39894228040143268) * exp_neg(A(0.5) * a * a)};
  }
  const A s = inverse(A(1) + exp_neg(a));                // 0 and 1 at the infinities
  if (act == EQT_ACT_SIGMOID) return {s, s * (A(1) - s)};
  return {a * s, s * (A(1) + a * (A(1) - s))};
}

int tensor_forward_f32(const GatedArgs& p, cudaStream_t s);         // gated_f32.cu and gated_bf16.cu, which compile side by side
int tensor_forward_bf16(const GatedArgs& p, cudaStream_t s);
int tensor_backward_f32(const GatedArgs& p, cudaStream_t s);
int tensor_backward_bf16(const GatedArgs& p, cudaStream_t s);
int tensor_form_f32(const GatedArgs& p, int product);                // eqt_gated_form
int tensor_form_bf16(const GatedArgs& p, int product);

}  // namespace gated
}  // namespace eqt
