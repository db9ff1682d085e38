// What the files of the gated layers (gated.cu, tc_gated.cu) share.
#pragma once
#include "igemm_problems.cuh"
#include "nrs_internal.h"

namespace gated {

// 1 / (1 + exp(-v)), and exp(-v) itself, kept finite.  The exponential as the hardware's power of two, 2 ulp, of -v log2(e)
// taken in two parts (its rounding error is put back to first order), and its reciprocal, 1 ulp: a third of the instructions
// that expf and a correctly rounded division take, which is what these element-wise passes were bound by.
// Below -kFar it is 0: exp(87) is the last whose reciprocal is a normal number, and a reciprocal held there instead would be
// multiplied by values of any size.  (A NaN comes out as 0 too, and through the product with it as itself.)
__device__ __forceinline__ float sigmoid(float v, float& e) {
  constexpr float kLog2e = 1.4426950408889634f, kRest = (float)(1.4426950408889634 - (double)kLog2e), kLn2 = 0.6931471805599453f, kFar = 87.0f;
  const float x = fmaxf(fminf(-v, kFar), -120.0f), t = x * kLog2e, rest = fmaf(x, kRest, fmaf(x, kLog2e, -t));
  float p, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(t));
  e = fmaf(p, rest * kLn2, p);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + e));
  return x < kFar ? s : 0.0f;
}
// act(a) and its derivative.  SiLU is a s with s = sigmoid(a), GELU (the tanh form) with s = sigmoid(2 u), u = sqrt(2/pi) (a +
// 0.044715 a^3); with w the sigmoid's argument the derivative is s + a s (1 - s) dw/da, and 1 - s = e s cancels nowhere.
__device__ __forceinline__ void act_both(float a, int kind, float& f, float& d) {
  if (kind == NRS_ACT_SILU || kind == NRS_ACT_GELU) {
    const float a2 = a * a;
    const float w = kind == NRS_ACT_SILU ? a : 1.5957691216f * a * fmaf(0.044715f, a2, 1.0f);
    const float dw = kind == NRS_ACT_SILU ? 1.0f : 1.5957691216f * fmaf(3.0f * 0.044715f, a2, 1.0f);
    float e;
    const float s = sigmoid(w, e);
    f = a * s;
    d = e > 0.0f ? fmaf(f * (e * s), s > 0.0f ? dw : 0.0f, s) : 1.0f;   // (e == 0, s == 0: a far out, where a dw may leave f32's range)
  } else if (kind == NRS_ACT_RELU) {
    f = a > 0.0f ? a : 0.0f;
    d = a > 0.0f ? 1.0f : 0.0f;
  } else {
    f = a;
    d = 1.0f;
  }
}
__device__ __forceinline__ float act(float a, int kind) {
  float f, d;
  act_both(a, kind, f, d);
  return f;
}

struct Shape { int m, n, k, act; };

}  // namespace gated

// The tensor-core forms (tc_gated.cu): f16 pairs, 3xTF32 mode; NRS_ERR_UNSUPPORTED (no error text) outside their range.
int nrs_tc_gated_fwd(nrs_ctx* ctx, const gated::Shape& s, const float* x, const float* w_gate, const float* w_up, float* h, float* pre_gate, float* pre_up);
int nrs_tc_gated_bwd(nrs_ctx* ctx, const gated::Shape& s, const float* x, const float* w_gate, const float* w_up, const float* pre_gate, const float* pre_up,
                     const float* dh, float* dx, float* dw_gate, float* dw_up, int acc_x, int acc_w);
// The forward pass of some dozen rows (gated_skinny.cu); NRS_ERR_UNSUPPORTED (no error text) likewise.
int nrs_gated_skinny_fwd(nrs_ctx* ctx, const gated::Shape& s, const float* x, const float* w_gate, const float* w_up, float* h, float* pre_gate, float* pre_up);
