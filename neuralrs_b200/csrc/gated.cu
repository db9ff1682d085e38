// Gated feed-forward layers, h = act(x Wg) . (x Wu), and their gradients: entry points, the form for a few rows, and the
// form of the FP32 and TF32 modes and of layers too small for the tensor cores.  No reference counterpart (its feed-forward
// is ungated, src/cuda/nn/transformer_block.rs:37-40).
//
// Up to 15 rows (tokens that are being generated; 5 and more of a large layer take gated_skinny.cu): bound by the weights, 8 k n
// bytes read once.  A block owns 32 columns of
// both matrices and a share of k; its warps read four rows of 128 bytes with each load of either matrix, four loads of each
// under way, against values of x in shared memory.  The shares of k are the CTAs of a cluster, which add their sums up
// through distributed shared memory: with 2752 columns there are 86 blocks of columns for 148 SMs.
#include <algorithm>

#include "gated.h"
#include "tc_common.cuh"

namespace {

using gated::Shape;

constexpr int kFewRows = 15, kThreads = 256, kWarps = kThreads / 32, kCols = 32, kStageK = 512;

// ROWS: rows of x at a time.  VEC: four columns a lane, four rows of the weights a warp; else a column and a row.
template <int ROWS, bool VEC>
__global__ void __launch_bounds__(kThreads)
gated_few_kernel(const float* __restrict__ x, const float* __restrict__ wg, const float* __restrict__ wu, float* __restrict__ h, float* __restrict__ pre_gate,
                 float* __restrict__ pre_up, int m, int n, int k, int act, int shares, int per_share) {
  NRS_PDL_PROLOGUE();
  constexpr int C = VEC ? 4 : 1, G = VEC ? 4 : 1;          // columns of a lane, weight rows of a warp's load
  __shared__ float xs[kStageK][ROWS];
  __shared__ float sums[2][ROWS][kCols];
  __shared__ float part[kWarps][2][ROWS][kCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = VEC ? lane >> 3 : 0, c = VEC ? (lane & 7) * 4 : lane;
  const int share = blockIdx.x % shares, n0 = blockIdx.x / shares * kCols, m0 = blockIdx.y * ROWS;
  const int k_begin = share * per_share, k_end = min(k, k_begin + per_share);
  const bool have = n0 + c < n;                            // (VEC: n is a multiple of 4)
  float acc[2][ROWS][C] = {};
  for (int kk = k_begin; kk < k_end; kk += kStageK) {
    const int rows = min(kStageK, k_end - kk);
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * kStageK; i += kThreads) {   // (k fast: whole lines of x)
      const int r = i / kStageK, j = i % kStageK;
      if (j < rows) xs[j][r] = m0 + r < m ? x[(size_t)(m0 + r) * k + kk + j] : 0.0f;
    }
    __syncthreads();
    constexpr int kDeep = 4;
    for (int j0 = warp * G + group; j0 < rows + group; j0 += kDeep * kWarps * G) {
      float a[kDeep][C], b[kDeep][C];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const int j = j0 + d * kWarps * G;
        const size_t at = (size_t)(kk + j) * n + n0 + c;
        const bool on = have && j < rows;
        if constexpr (VEC) {
          const float4 p = on ? *reinterpret_cast<const float4*>(wg + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          const float4 q = on ? *reinterpret_cast<const float4*>(wu + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          a[d][0] = p.x; a[d][1] = p.y; a[d][2] = p.z; a[d][3] = p.w;
          b[d][0] = q.x; b[d][1] = q.y; b[d][2] = q.z; b[d][3] = q.w;
        } else {
          a[d][0] = on ? wg[at] : 0.0f;
          b[d][0] = on ? wu[at] : 0.0f;
        }
      }
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const int j = j0 + d * kWarps * G;
        if (j >= rows) continue;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float v = xs[j][r];
#pragma unroll
          for (int e = 0; e < C; ++e) {
            acc[0][r][e] = fmaf(v, a[d][e], acc[0][r][e]);
            acc[1][r][e] = fmaf(v, b[d][e], acc[1][r][e]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int e = 0; e < C; ++e) {
        float v = acc[s][r][e];
        if (VEC) {
          v += __shfl_xor_sync(0xffffffffu, v, 8);
          v += __shfl_xor_sync(0xffffffffu, v, 16);
        }
        if (group == 0) part[warp][s][r][c + e] = v;
      }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * ROWS * kCols; i += kThreads) {
    const int s = i / (ROWS * kCols), r = i / kCols % ROWS, cc = i % kCols;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += part[w][s][r][cc];
    sums[s][r][cc] = v;
  }
  if (shares > 1) tc::cluster_sync(); else __syncthreads();
  // Each CTA of the cluster finishes its share of the results, adding the others' sums in their order.
  for (int i = threadIdx.x * shares + share; i < ROWS * kCols; i += kThreads * shares) {
    const int r = i / kCols, cc = i % kCols;
    if (m0 + r >= m || n0 + cc >= n) continue;
    float a = 0.0f, u = 0.0f;
    if (shares == 1) {
      a = sums[0][r][cc];
      u = sums[1][r][cc];
    } else {
      for (int s = 0; s < shares; ++s) {
        float p, q;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(tc::cluster_addr(&sums[0][r][cc], s)));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(q) : "r"(tc::cluster_addr(&sums[1][r][cc], s)));
        a += p;
        u += q;
      }
    }
    const size_t at = (size_t)(m0 + r) * n + n0 + cc;
    if (pre_gate) { pre_gate[at] = a; pre_up[at] = u; }
    h[at] = gated::act(a, act) * u;
  }
  if (shares > 1) tc::cluster_sync();                      // (nobody leaves while its sums are read)
}

int few_rows(nrs_ctx* ctx, const Shape& s, const float* x, const float* wg, const float* wu, float* h, float* pg, float* pu) {
  const bool vec = s.n % 4 == 0 && (((uintptr_t)wg | (uintptr_t)wu) & 15) == 0;
  const int blocks = (s.n - 1) / kCols + 1;   // (n up to the last that an int counts)
  int shares = 1;   // until there are two blocks an SM, or a share of k is two loads of a warp
  while (shares < 8 && blocks * shares < 2 * ctx->sm_count && s.k / (2 * shares) >= 256) shares *= 2;
  const int per = (s.k + shares - 1) / shares;
  const int rows = s.m == 1 ? 1 : s.m == 2 ? 2 : s.m <= 4 ? 4 : 8;
  const dim3 grid((unsigned)(blocks * shares), (unsigned)((s.m + rows - 1) / rows));
#define NRS_FEW(R_, V_)                                                                                                                                  \
  (void)nrs_pdl_launch_cluster((unsigned)shares, gated_few_kernel<R_, V_>, grid, dim3(kThreads), (size_t)0, ctx->stream, x, wg, wu, h, pg, pu, s.m, s.n, \
                               s.k, s.act, shares, per)
#define NRS_FEW_ROWS(V_)                       \
  switch (rows) {                              \
    case 1: NRS_FEW(1, V_); break;             \
    case 2: NRS_FEW(2, V_); break;             \
    case 4: NRS_FEW(4, V_); break;             \
    default: NRS_FEW(8, V_); break;            \
  }
  if (vec) { NRS_FEW_ROWS(true) } else { NRS_FEW_ROWS(false) }
#undef NRS_FEW_ROWS
#undef NRS_FEW
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

// Where the tensor-core form without a pass over the weights is the fastest (us; few rows, that one, staged operands).  Up to 4
// rows stay in f32 and one launch: ahead on smaller layers; with the weights out of L2 a tenth behind at 2048 x 5504 and a sixth at
// 8192 x 5504.
//   rows  k x n         few   this  staged        rows  k x n        this  staged
//   4     2048 x 5504   25.0  24.1                 16   2048 x 5504   24.9  78.4
//   8     2048 x 5504   55.2  24.7                128   2048 x 5504   52.8  80.1
//   8     1024 x 2752   15.9  11.3                200   2048 x 5504   98.6  92.6
//   8     2048 x 700    10.0   9.9                128   256 x 1024     9.3  12.7
//   8     512 x 1000     7.2   7.2                 32   100 x 5000    10.8  11.8
//   8     100 x 5000     6.2   9.8                 64   100 x 5000    13.6  12.1
bool skinny(const Shape& s) {
  if (s.m <= kFewRows) return s.m > 4 && (double)s.m * s.n * s.k >= 8e6;
  return s.m <= 32 || (s.m <= 128 && s.k >= 256);
}

// h = act(a) u, element by element.
__global__ void __launch_bounds__(256) gated_act_kernel(const float* __restrict__ a, const float* __restrict__ u, float* __restrict__ h, size_t total, int act) {
  NRS_PDL_PROLOGUE();
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) h[i] = gated::act(a[i], act) * u[i];
}
// da = dh u act'(a), du = dh act(a)
__global__ void __launch_bounds__(256)
gated_act_bwd_kernel(const float* __restrict__ g, const float* __restrict__ a, const float* __restrict__ u, float* __restrict__ da, float* __restrict__ du,
                     size_t total, int act) {
  NRS_PDL_PROLOGUE();
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
    float f, d;
    gated::act_both(a[i], act, f, d);
    da[i] = g[i] * u[i] * d;
    du[i] = g[i] * f;
  }
}

unsigned grid_for(const nrs_ctx* ctx, size_t total) { return (unsigned)std::min<size_t>((total + 255) / 256, (size_t)ctx->sm_count * 16); }

// Two [m][n] blocks of the context's scratch.
int two_blocks(nrs_ctx* ctx, const Shape& s, float** a, float** b) {
  const size_t each = ((size_t)s.m * s.n + 63) / 64 * 64;
  void* p = nullptr;
  const int st = nrs_ws_slot(ctx, NRS_WS_GATED, 2 * each * sizeof(float), &p);
  *a = (float*)p;
  *b = *a + each;
  return st;
}

int check_shape(nrs_ctx* ctx, const char* who, int m, int n, int k, int act) {
  NRS_REQUIRE(ctx, m >= 0 && n >= 0 && k >= 0, NRS_ERR_SHAPE, "%s: negative dimension", who);
  NRS_REQUIRE(ctx, act >= NRS_ACT_NONE && act <= NRS_ACT_SILU, NRS_ERR_ARG, "%s: unknown activation %d", who, act);
  return NRS_OK;
}

}  // namespace

extern "C" {

int nrs_gated_linear_fwd(nrs_ctx* ctx, const float* x, const float* w_gate, const float* w_up, float* h, float* pre_gate, float* pre_up, int m, int n, int k,
                         int act) {
  NRS_REQUIRE_CTX(ctx);
  int st = check_shape(ctx, __func__, m, n, k, act);
  if (st != NRS_OK || m == 0 || n == 0) return st;
  NRS_REQUIRE(ctx, h && (k == 0 || (x && w_gate && w_up)), NRS_ERR_ARG, "%s: null tensor", __func__);
  NRS_REQUIRE(ctx, (pre_gate != nullptr) == (pre_up != nullptr), NRS_ERR_ARG, "%s: both projections are kept, or neither", __func__);
  NrsDeviceGuard on(ctx);
  if (k == 0) {   // empty sums
    const size_t bytes = (size_t)m * n * sizeof(float);
    for (float* p : {h, pre_gate, pre_up})
      if (p && (st = nrs_memset_zero(ctx, p, bytes)) != NRS_OK) return st;
    return NRS_OK;
  }
  const Shape s{m, n, k, act};
  if (skinny(s)) {
    st = nrs_gated_skinny_fwd(ctx, s, x, w_gate, w_up, h, pre_gate, pre_up);
    if (st != NRS_ERR_UNSUPPORTED) return st;
  }
  if (m <= kFewRows) return few_rows(ctx, s, x, w_gate, w_up, h, pre_gate, pre_up);
  st = nrs_tc_gated_fwd(ctx, s, x, w_gate, w_up, h, pre_gate, pre_up);
  if (st != NRS_ERR_UNSUPPORTED) return st;
  float *a = pre_gate, *u = pre_up;
  if (!a && (st = two_blocks(ctx, s, &a, &u)) != NRS_OK) return st;
  st = nrs_gemm(ctx, 0, 0, m, n, k, x, w_gate, a, nullptr, NRS_ACT_NONE, 0.0f);
  if (st == NRS_OK) st = nrs_gemm(ctx, 0, 0, m, n, k, x, w_up, u, nullptr, NRS_ACT_NONE, 0.0f);
  if (st != NRS_OK) return st;
  NRS_PDL_LAUNCH(gated_act_kernel, grid_for(ctx, (size_t)m * n), 256, 0, ctx->stream, a, u, h, (size_t)m * n, act);
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

int nrs_gated_linear_bwd(nrs_ctx* ctx, const float* x, const float* w_gate, const float* w_up, const float* pre_gate, const float* pre_up, const float* dh,
                         float* dx, float* dw_gate, float* dw_up, int m, int n, int k, int act, int accumulate_x, int accumulate_w) {
  NRS_REQUIRE_CTX(ctx);
  int st = check_shape(ctx, __func__, m, n, k, act);
  if (st != NRS_OK || k == 0) return st;
  NRS_REQUIRE(ctx, (dw_gate != nullptr) == (dw_up != nullptr), NRS_ERR_ARG, "%s: both weights' gradients are asked for, or neither", __func__);
  NrsDeviceGuard on(ctx);
  if (m == 0 || n == 0) {   // empty sums
    if (dx && m > 0 && !accumulate_x) st = nrs_memset_zero(ctx, dx, (size_t)m * k * sizeof(float));
    for (float* p : {dw_gate, dw_up})
      if (st == NRS_OK && p && n > 0 && !accumulate_w) st = nrs_memset_zero(ctx, p, (size_t)k * n * sizeof(float));
    return st;
  }
  if (!dx && !dw_gate) return NRS_OK;
  NRS_REQUIRE(ctx, pre_gate && pre_up && dh && (!dx || (w_gate && w_up)) && (!dw_gate || x), NRS_ERR_ARG, "%s: null tensor", __func__);
  const Shape s{m, n, k, act};
  st = nrs_tc_gated_bwd(ctx, s, x, w_gate, w_up, pre_gate, pre_up, dh, dx, dw_gate, dw_up, accumulate_x != 0, accumulate_w != 0);
  if (st != NRS_ERR_UNSUPPORTED) return st;
  float *da = nullptr, *du = nullptr;
  if ((st = two_blocks(ctx, s, &da, &du)) != NRS_OK) return st;
  NRS_PDL_LAUNCH(gated_act_bwd_kernel, grid_for(ctx, (size_t)m * n), 256, 0, ctx->stream, dh, pre_gate, pre_up, da, du, (size_t)m * n, act);
  NRS_LAUNCHED(ctx);
  if (dx) {
    st = nrs_gemm(ctx, 0, 1, m, k, n, da, w_gate, dx, nullptr, NRS_ACT_NONE, accumulate_x ? 1.0f : 0.0f);
    if (st == NRS_OK) st = nrs_gemm(ctx, 0, 1, m, k, n, du, w_up, dx, nullptr, NRS_ACT_NONE, 1.0f);
    if (st != NRS_OK) return st;
  }
  if (dw_gate) {
    st = nrs_gemm(ctx, 1, 0, k, n, m, x, da, dw_gate, nullptr, NRS_ACT_NONE, accumulate_w ? 1.0f : 0.0f);
    if (st == NRS_OK) st = nrs_gemm(ctx, 1, 0, k, n, m, x, du, dw_up, nullptr, NRS_ACT_NONE, accumulate_w ? 1.0f : 0.0f);
    if (st != NRS_OK) return st;
  }
  return NRS_OK;
}

}  // extern "C"
