// Gated feed-forward layers on the tensor cores:  h = act(x Wg) . (x Wu)  in one kernel, and its gradients
//   da = dh . u act'(a),  du = dh . act(a)        (a = x Wg, u = x Wu, as the forward pass left them)
//   dx = da Wg^T + du Wu^T,   dWg = x^T da,   dWu = x^T du
// in three: the elementwise part, which writes da and du as operand planes side by side and nothing else; one product over
// both for dx (the reduction runs through the columns of da, then of du); one for both weight gradients.
//
// Main loop: tc_mainloop.cuh, f16 pairs (3xTF32), chains of 256 values of K summed in registers.  Forward, a tile's 128
// columns are 64 of a and the same 64 of u, so a warp that has both in its registers multiplies them where they are: neither
// leaves the SM unless the backward pass needs it.  (A pair of CTAs brings the 64 rows of Wg^T in one and of Wu^T in the
// other.)
#include "gated.h"
#include "tc_mainloop.cuh"

namespace {

using gated::Shape;

enum Product { kForward, kInput, kWeights };

template <Product P>
struct GatedPolicy {
  static constexpr bool kCanEmit = false, kConv = false, kSlab = false;
  static constexpr bool kGated = P == kForward, kAMnMajor = P == kWeights, kBMnMajor = P == kWeights;
  static constexpr bool kMaySplit = P != kForward;
  static constexpr int kEpiWarps = 16, kTeamWarps = 4;
  static constexpr int kChainK = 256;
  int order() const { return tc::kRaster; }

  float* out[2];         // forward: h; input: dx; weights: dWg, dWu
  float* pre[2];         // forward: a, u, or null
  int M, N;              // of the output as it is stored (weights: of one matrix)
  int ld;                // weights: columns of one matrix in the product, padding included; input: columns of da, likewise
  int act, accumulate;
  bool vec;              // rows of the outputs start on 16 bytes

  __device__ __forceinline__ bool clip(int, int, int, int*, int*) const { return true; }
  __device__ __forceinline__ uint32_t a_slice_rows() const { return tc::BM; }
  struct Cursor { int col, row, mat; };
  template <int KW>
  __device__ __forceinline__ Cursor cursor(int tile_m, int, int kb) const {
    const int col = kb * KW;
    if (P == kInput && col >= ld) return Cursor{col - ld, tile_m * tc::BM, 1};
    return Cursor{col, tile_m * tc::BM, 0};
  }
  template <int KW>
  __device__ __forceinline__ void advance(Cursor& c) const {
    c.col += KW;
    if (P == kInput && c.col == ld) { c.col = 0; c.mat = 1; }
  }
  template <bool PAIR, int KW, int ROW_BYTES>
  __device__ __forceinline__ void load_a(void* dst, const CUtensorMap* tm, uint32_t bar, const Cursor& c) const {
    if (P == kWeights) tc::tma_load_3d_to<PAIR>(dst, tm, bar, 0, c.col, c.row / KW);
    else tc::tma_load_3d_to<PAIR>(dst, tm, bar, c.col, c.row, c.mat);
  }
  template <int BN, bool PAIR, int KW, int ROW_BYTES>
  __device__ __forceinline__ void load_b(void* dst, const CUtensorMap* tm, uint32_t bar, const Cursor& c, int n0) const {
    if (P == kWeights) {
      tc::tma_load_3d_to<PAIR>(dst, tm, bar, 0, c.col, n0 / KW);
    } else if (P == kInput) {
      tc::tma_load_3d_to<PAIR>(dst, tm, bar, c.col, n0, c.mat);
    } else if (PAIR) {           // half of the tile's columns: this CTA's matrix
      tc::tma_load_3d_to<PAIR>(dst, tm, bar, c.col, n0 / BN * (BN / 2), n0 % BN != 0);
    } else {
      tc::tma_load_3d_to<PAIR>(dst, tm, bar, c.col, n0 / 2, 0);
      tc::tma_load_3d_to<PAIR>(reinterpret_cast<uint8_t*>(dst) + BN / 2 * ROW_BYTES, tm, bar, c.col, n0 / 2, 1);
    }
  }
  __device__ __forceinline__ float out_bound(float, float, int) const { return 0.0f; }
  __device__ __forceinline__ int row(int, int, int) const { return 0; }
  template <int W>
  __device__ __forceinline__ int fetch(int, int, bool) const { return 0; }

  // Forward: a warp's 32 rows of 16 columns of a (sums[0]) and of u (sums[1]).
  template <int MINE>
  __device__ __forceinline__ void finish(int tile_m, int tile_n, int c, int r0, int lane, float* scratch, float (&sums)[MINE][16], uint32_t&) const {
    static_assert(MINE == 2, "the columns of both matrices");
    const int n = tile_n * 64 + c * 16 + (lane & 3) * 4, m0 = tile_m * tc::BM + r0, left = N - n;
    if (tile_n * 64 + c * 16 >= N) return;
    uint32_t r[16];
    float4 v[4];
    auto send = [&](float* dst) {
      tc::rows_to_lines(scratch, lane, r, v);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (m0 + 8 * i < M) tc::store_guarded(dst + (size_t)(m0 + 8 * i) * N + n, v[i], left, vec);
    };
    if (pre[0]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(sums[s][j]);
        send(pre[s]);
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(gated::act(sums[0][j], act) * sums[1][j]);
    send(out[0]);
  }

  // Four row segments of the output, rows r0 + 8 i of the tile, columns n..n+3.
  __device__ __forceinline__ void epilogue(int tile_m, int r0, int n, const float4 (&v)[4]) const {
    const int mat = P == kWeights && n >= ld ? 1 : 0, c = n - mat * ld, left = N - c, m0 = tile_m * tc::BM + r0;
    if (left <= 0) return;
    float* dst = out[mat] + (size_t)m0 * N + c;
#pragma unroll
    for (int i = 0; i < 4; ++i, dst += (size_t)8 * N) {
      if (m0 + 8 * i >= M) return;
      float4 q = v[i];
      if (accumulate) {
        const float4 o = tc::load_guarded(dst, left, vec);
        q = make_float4(o.x + q.x, o.y + q.y, o.z + q.z, o.w + q.w);
      }
      tc::store_guarded(dst, q, left, vec);
    }
  }
  // One element, from the pass that sums a K-split.
  template <bool SPLIT>
  __device__ __forceinline__ void store(int tile_m, int, int row, int n, float v, float, uint32_t&) const {
    const int mat = P == kWeights && n >= ld ? 1 : 0, c = n - mat * ld, m = tile_m * tc::BM + row;
    if (m >= M || c >= N) return;
    float* dst = out[mat] + (size_t)m * N + c;
    *dst = accumulate ? *dst + v : v;
  }
};

// ------------------------------------------------------------------------------------------------ da and du

// Four values of da and du.
__device__ __forceinline__ void gradients(float4 g, float4 a, float4 u, int kind, float4& da, float4& du) {
  const float gg[4] = {g.x, g.y, g.z, g.w}, aa[4] = {a.x, a.y, a.z, a.w}, uu[4] = {u.x, u.y, u.z, u.w};
  float p[4], q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float f, d;
    gated::act_both(aa[j], kind, f, d);
    p[j] = gg[j] * uu[j] * d;
    q[j] = gg[j] * f;
  }
  da = make_float4(p[0], p[1], p[2], p[3]);
  du = make_float4(q[0], q[1], q[2], q[3]);
}

// Two passes over dh, a and u: the largest magnitude of what they give (WRITE == false), then the pairs
// [m][da: ld | du: ld], zeros from n to ld.
template <bool WRITE>
__global__ void __launch_bounds__(256)
gated_planes_kernel(const float* __restrict__ g, const float* __restrict__ a, const float* __restrict__ u, float* hi, float* lo, NrsRange* range, int m, int n,
                    int ld, NrsFastDiv div /*of ld / 4*/, int kind, bool vec) {
  NRS_PDL_PROLOGUE();
  const uint32_t quads = (uint32_t)m * (uint32_t)(ld / 4), stride = gridDim.x * blockDim.x;   // (the launcher checks the range)
  float scale = 1.0f;
  if (WRITE) {
    const float bound = range->top;
    scale = pr::scale_of(bound);
    if (blockIdx.x == 0 && threadIdx.x == 0) range->bound = bound;
  }
  uint32_t top = 0;
  constexpr int kDeep = 2;
  for (uint32_t i0 = blockIdx.x * blockDim.x + threadIdx.x; i0 < quads; i0 += kDeep * stride) {
    float4 vg[kDeep], va[kDeep], vu[kDeep];
    uint32_t row[kDeep], q[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const uint32_t i = i0 + k * stride;
      vg[k] = va[k] = vu[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i >= quads) continue;
      div.divmod(i, row[k], q[k]);
      const int left = n - (int)(4 * q[k]);
      if (left <= 0) continue;
      const size_t at = (size_t)row[k] * n + 4 * q[k];
      vg[k] = tc::load_guarded(g + at, left, vec);
      va[k] = tc::load_guarded(a + at, left, vec);
      vu[k] = tc::load_guarded(u + at, left, vec);
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      if (i0 + k * stride >= quads) continue;
      float4 da, du;
      gradients(vg[k], va[k], vu[k], kind, da, du);
      if (WRITE) {
        const size_t at = (size_t)row[k] * (2 * ld) + 4 * q[k];
        pr::put4(hi, lo, at, da, scale);
        pr::put4(hi, lo, at + ld, du, scale);
      } else {
        top = pr::seen4(top, da);
        top = pr::seen4(top, du);
      }
    }
  }
  if (!WRITE) {
    __syncwarp();
    pr::report(range, top);
  }
}

struct Planes {
  void *hi, *lo;
  const NrsRange* range;
};

int round64(int v) { return (v + 63) / 64 * 64; }

// [batch][rows][cols] planes with rows ld values apart, cols values of K a row.
bool map_k(CUtensorMap* t, const void* base, int cols, int rows, int batch, size_t ld, size_t bstride, int box_rows) {
  const uint64_t dim[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)batch}, str[2] = {ld, bstride};
  const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
  return tc::encode_tmap(t, base, true, 3, dim, str, box);
}
// Rows of K: [row block of 64 columns][k][64].
bool map_mn(CUtensorMap* t, const void* base, int cols /*a multiple of 64*/, int k, int box_cols) {
  const uint64_t dim[3] = {64, (uint64_t)k, (uint64_t)(cols / 64)}, str[2] = {(uint64_t)cols, 64};
  const uint32_t box[3] = {64, 64, (uint32_t)(box_cols / 64)};
  return tc::encode_tmap(t, base, true, 3, dim, str, box, true);
}

template <int BN, bool PAIR, Product P>
int run(nrs_ctx* ctx, const Planes& A, const Planes& B, const GatedPolicy<P>& pol, int rows, int cols, int kdim, int a_batch, size_t a_ld, size_t a_stride,
        int b_rows, size_t b_ld, size_t b_stride, int kblocks) {
  constexpr int kBRows = PAIR || P == kForward ? BN / 2 : BN;   // rows of B in one load
  CUtensorMap a[2], b[2];
  bool ok = true;
  for (int i = 0; i < 2; ++i) {
    const void *pa = i ? A.lo : A.hi, *pb = i ? B.lo : B.hi;
    if (P == kWeights) ok = ok && map_mn(&a[i], pa, (int)a_ld, kdim, tc::BM) && map_mn(&b[i], pb, (int)b_ld, kdim, kBRows);
    else ok = ok && map_k(&a[i], pa, kdim, rows, a_batch, a_ld, a_stride, tc::BM) && map_k(&b[i], pb, kdim, b_rows, 2, b_ld, b_stride, kBRows);
  }
  NRS_REQUIRE(ctx, ok, NRS_ERR_CUDA, "gated layer: cuTensorMapEncodeTiled failed (%d x %d x %d)", rows, cols, kdim);
  return tc::launch<BN, 2, PAIR, 64, GatedPolicy<P>>(ctx, a[0], a[1], b[0], b[1], pol, (rows + tc::BM - 1) / tc::BM, cols, 1, kblocks,
                                                     tc::Ranges{A.range, B.range, nullptr});
}

bool aligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}

// Planes of x [m][k] with rows round64(k) values apart.
int stage_x(nrs_ctx* ctx, const Shape& s, const float* x, Planes* out) {
  const int ld = round64(s.k);
  int st = nrs_ws_planes(ctx, NRS_WS_A, (size_t)s.m * ld, true, &out->hi, &out->lo);
  if (st == NRS_OK) st = nrs_tc_stage(ctx, x, (float*)out->hi, (float*)out->lo, s.m, s.k, ld, 1, 0, 0, false);
  out->range = nrs_range_of(ctx, out->hi);
  return st;
}
// Planes of both weights, one behind the other, with one range: transposed ([n][k]), or as stored ([k][n]).
int stage_weights(nrs_ctx* ctx, const Shape& s, const float* wg, const float* wu, bool transposed, Planes* out) {
  const float* w[2] = {wg, wu};
  const int rows = transposed ? s.n : s.k, cols = transposed ? s.k : s.n, ld = round64(cols);
  int st = nrs_ws_planes(ctx, NRS_WS_B, 2 * (size_t)rows * ld, true, &out->hi, &out->lo);
  if (st == NRS_OK) st = nrs_tc_stage_each(ctx, w, 2, (float*)out->hi, (float*)out->lo, rows, cols, ld, (size_t)rows * ld, transposed);
  out->range = nrs_range_of(ctx, out->hi);
  return st;
}

bool applies(const nrs_ctx* ctx, const Shape& s) {
  // (from 16 rows on, as the ungated products; the elementwise passes count quads in 32 bits)
  return ctx->math_mode == NRS_MATH_3XTF32 && tc::tensor_map_encoder() && s.m >= 16 && s.n >= 32 && s.k >= 32 &&
         (uint64_t)s.m * (uint64_t)(round64(s.n) / 4) < 0x40000000ull && s.n <= (1 << 24) && s.k <= (1 << 24);
}

}  // namespace

int nrs_tc_gated_fwd(nrs_ctx* ctx, const Shape& s, const float* x, const float* w_gate, const float* w_up, float* h, float* pre_gate, float* pre_up) {
  if (!applies(ctx, s)) return NRS_ERR_UNSUPPORTED;
  Planes A{}, B{};
  int st = stage_x(ctx, s, x, &A);
  if (st == NRS_OK) st = stage_weights(ctx, s, w_gate, w_up, true, &B);
  if (st != NRS_OK) return st;
  GatedPolicy<kForward> pol{};
  pol.out[0] = h; pol.pre[0] = pre_gate; pol.pre[1] = pre_up;
  pol.M = s.m; pol.N = s.n; pol.act = s.act;
  pol.vec = s.n % 4 == 0 && aligned({h, pre_gate, pre_up});
  NrsProfScope prof(ctx, NRS_PROF_GEMM, 4.0 * s.m * s.n * s.k);
  const int ld = round64(s.k), cols = 2 * round64(s.n), kb = ld / 64;
  // Pairs take 395 clocks per 32 values of K a round of 74, single tiles 530 a round of 148 (plan_tile's table).
  const long tm = (s.m + 127) / 128, tn = cols / 128, sms = ctx->sm_count;
  const long pairs = ((tm + 1) / 2 * tn + sms / 2 - 1) / (sms / 2) * 395, singles = (tm * tn + sms - 1) / sms * 530;
  if (pairs <= singles) return run<128, true, kForward>(ctx, A, B, pol, s.m, cols, s.k, 1, ld, (size_t)s.m * ld, s.n, ld, (size_t)s.n * ld, kb);
  return run<128, false, kForward>(ctx, A, B, pol, s.m, cols, s.k, 1, ld, (size_t)s.m * ld, s.n, ld, (size_t)s.n * ld, kb);
}

int nrs_tc_gated_bwd(nrs_ctx* ctx, const Shape& s, const float* x, const float* w_gate, const float* w_up, const float* pre_gate, const float* pre_up,
                     const float* dh, float* dx, float* dw_gate, float* dw_up, int acc_x, int acc_w) {
  if (!applies(ctx, s)) return NRS_ERR_UNSUPPORTED;
  const int ldn = round64(s.n), ldk = round64(s.k);
  Planes D{};
  int st = nrs_ws_planes(ctx, NRS_WS_GATED, 2 * (size_t)s.m * ldn, true, &D.hi, &D.lo);
  if (st != NRS_OK) return st;
  NrsRange* range = nullptr;
  st = nrs_range_renew(ctx, D.hi, &range);
  if (st != NRS_OK) return st;
  D.range = range;
  const bool vec = s.n % 4 == 0 && aligned({dh, pre_gate, pre_up});
  const uint32_t quads = (uint32_t)s.m * (uint32_t)(ldn / 4);
  const unsigned blocks = std::min<unsigned>((quads + 511) / 512, (unsigned)ctx->sm_count * 8);
  NRS_PDL_LAUNCH(gated_planes_kernel<false>, blocks, 256, 0, ctx->stream, dh, pre_gate, pre_up, (float*)D.hi, (float*)D.lo, range, s.m, s.n, ldn,
                 NrsFastDiv(ldn / 4), s.act, vec);
  NRS_LAUNCHED(ctx);
  NRS_PDL_LAUNCH(gated_planes_kernel<true>, blocks, 256, 0, ctx->stream, dh, pre_gate, pre_up, (float*)D.hi, (float*)D.lo, range, s.m, s.n, ldn,
                 NrsFastDiv(ldn / 4), s.act, vec);
  NRS_LAUNCHED(ctx);
  const size_t ld2 = 2 * (size_t)ldn;
  if (dx) {
    Planes W{};
    st = stage_weights(ctx, s, w_gate, w_up, false, &W);
    if (st != NRS_OK) return st;
    GatedPolicy<kInput> pol{};
    pol.out[0] = dx; pol.M = s.m; pol.N = s.k; pol.ld = ldn; pol.accumulate = acc_x;
    pol.vec = s.k % 4 == 0 && aligned({dx});
    NrsProfScope prof(ctx, NRS_PROF_GEMM, 4.0 * s.m * s.n * s.k);
    const tc::TilePlan t = tc::plan_tile(ctx, (s.m + 127) / 128, s.k, 1, 2 * ldn / 32, true, 0.004, false, false);
#define NRS_RUN(BN_, PAIR_) run<BN_, PAIR_, kInput>(ctx, D, W, pol, s.m, s.k, s.n, 2, ld2, ldn, s.k, ldn, (size_t)s.k * ldn, 2 * ldn / 64)
    st = t.bn == 128 ? (t.pair ? NRS_RUN(128, true) : NRS_RUN(128, false)) : (t.pair ? NRS_RUN(64, true) : NRS_RUN(64, false));
#undef NRS_RUN
    if (st != NRS_OK) return st;
  }
  if (dw_gate || dw_up) {
    Planes X{};
    st = stage_x(ctx, s, x, &X);
    if (st != NRS_OK) return st;
    GatedPolicy<kWeights> pol{};
    pol.out[0] = dw_gate; pol.out[1] = dw_up; pol.M = s.k; pol.N = s.n; pol.ld = ldn; pol.accumulate = acc_w;
    pol.vec = s.n % 4 == 0 && aligned({dw_gate, dw_up});
    NrsProfScope prof(ctx, NRS_PROF_GEMM, 4.0 * s.m * s.n * s.k);
    const tc::TilePlan t = tc::plan_tile(ctx, (s.k + 127) / 128, 2 * ldn, 1, (s.m + 31) / 32, true, 0.004, false, false);
#define NRS_RUN(BN_, PAIR_) run<BN_, PAIR_, kWeights>(ctx, X, D, pol, s.k, 2 * ldn, s.m, 1, ldk, 0, 0, ld2, 0, (s.m + 63) / 64)
    // (columns of 64 in a CTA's share of B: no pair of 64)
    st = t.bn == 128 && t.pair ? NRS_RUN(128, true) : t.bn == 128 ? NRS_RUN(128, false) : NRS_RUN(64, false);
#undef NRS_RUN
    if (st != NRS_OK) return st;
  }
  return NRS_OK;
}
