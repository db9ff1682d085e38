// What the files of the gated layers (gated.cu, tc_gated.cu) share.
#pragma once
#include "igemm_problems.cuh"
#include "nrs_internal.h"

namespace gated {

// exp(-a), kept finite
__device__ __forceinline__ float exp_minus(float a) { return expf(fminf(-a, 80.0f)); }

__device__ __forceinline__ float act(float a, int kind) {
  if (kind == NRS_ACT_SILU) return a / (1.0f + exp_minus(a));
  return nrs_apply_act(a, kind);
}
// act(a) and its derivative.  SiLU: s (1 + a (1 - s)) with s = 1 / (1 + e), e = exp(-a), and 1 - s = e s, which cancels
// nowhere.
__device__ __forceinline__ void act_both(float a, int kind, float& f, float& d) {
  if (kind == NRS_ACT_SILU) {
    const float e = exp_minus(a), s = 1.0f / (1.0f + e);
    f = a * s;
    d = s * fmaf(a, e * s, 1.0f);
  } else if (kind == NRS_ACT_GELU) {
    f = nrs_gelu_f(a);
    d = nrs_gelu_d(a);
  } else if (kind == NRS_ACT_RELU) {
    f = a > 0.0f ? a : 0.0f;
    d = a > 0.0f ? 1.0f : 0.0f;
  } else {
    f = a;
    d = 1.0f;
  }
}

struct Shape { int m, n, k, act; };

}  // namespace gated

// The tensor-core forms (tc_gated.cu): f16 pairs, 3xTF32 mode; NRS_ERR_UNSUPPORTED (no error text) outside their range.
int nrs_tc_gated_fwd(nrs_ctx* ctx, const gated::Shape& s, const float* x, const float* w_gate, const float* w_up, float* h, float* pre_gate, float* pre_up);
int nrs_tc_gated_bwd(nrs_ctx* ctx, const gated::Shape& s, const float* x, const float* w_gate, const float* w_up, const float* pre_gate, const float* pre_up,
                     const float* dh, float* dx, float* dw_gate, float* dw_up, int acc_x, int acc_w);
