// Gated feed-forward layers on the tensor cores:  h = act(x Wg) . (x Wu)  in one kernel, and its gradients
//   da = dh . u act'(a),  du = dh . act(a)        (a = x Wg, u = x Wu, as the forward pass left them)
//   dx = da Wg^T + du Wu^T,   dWg = x^T da,   dWu = x^T du
// in three: the elementwise part, which writes da and du as operand planes side by side and nothing else; one product over
// both for dx (the reduction runs through the columns of da, then of du); one for both weight gradients.
//
// Main loop: tc_mainloop.cuh, f16 pairs (3xTF32), chains of 256 values of K summed in registers.  Forward, a tile's 128
// columns are 64 of a and the same 64 of u, so a warp that has both in its registers multiplies them where they are: neither
// leaves the SM unless the backward pass needs it.  (Of a pair of CTAs, one brings the columns of Wg and one those of Wu.)
//
// Operand planes: every tensor as it is stored, rows padded with zeros to a multiple of 64 values, Wg and Wu (da and du) side
// by side in one row.  The forward product reads the weights' planes with k across the rows, dx along them, the weight
// gradients x and da|du across: nothing is transposed (staging 2048 x 5504 weights transposed took 112 us, as they are 36).
// All of a pass's operands are measured by one launch and written by another.
//
// Every matrix has an exponent of its own, also where two lie side by side: a and u, dWg and dWu are results apart, and what is
// small in one of them is not to lose bits to the other.  dx adds da Wg^T and du Wu^T in one accumulator, so there the
// exponents of Wg and Wu are chosen such that both products carry the same one, that of the larger product: the other gives
// up only what lies below the sum's own bits.
#include "gated.h"
#include "tc_mainloop.cuh"

namespace {

using gated::Shape;

enum Product { kForward, kInput, kWeights };

template <Product P>
struct GatedPolicy {
  static constexpr bool kCanEmit = false, kConv = false, kSlab = false;
  static constexpr bool kGated = P == kForward, kAMnMajor = P == kWeights, kBMnMajor = P != kInput;
  static constexpr bool kMaySplit = P != kForward;
  static constexpr int kEpiWarps = 16, kTeamWarps = 4;
  static constexpr int kChainK = 256;
  int order() const { return tc::kRaster; }

  float* out[2];         // forward: h; input: dx; weights: dWg, dWu
  float* pre[2];         // forward: a, u, or null
  int M, N;              // of the output as it is stored (weights: of one matrix)
  int ld;                // n, padded: columns of one of the two matrices side by side
  const NrsRange *ra, *rb;   // of A's and B's matrices
  int act, accumulate;
  bool vec;              // rows of the outputs start on 16 bytes
  bool independent;      // of the kernel launched before it

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
      tc::tma_load_3d_to<PAIR>(dst, tm, bar, 0, c.col, n0 / BN + (n0 % BN != 0 ? ld / 64 : 0));
    } else {
      tc::tma_load_3d_to<PAIR>(dst, tm, bar, 0, c.col, n0 / BN);
      tc::tma_load_3d_to<PAIR>(reinterpret_cast<uint8_t*>(dst) + BN / 2 * ROW_BYTES, tm, bar, 0, c.col, n0 / BN + ld / 64);
    }
  }
  __device__ __forceinline__ float out_bound(float, float, int) const { return 0.0f; }
  // Both operands' exponents in the sums that belong to matrix `mat`; and which one a warp's i-th block, at column n, belongs to.
  __device__ __forceinline__ int exponents(int mat) const {
    if (P == kInput) return min(pr::scale_exp(ra[0].top) + pr::scale_exp(rb[0].top), pr::scale_exp(ra[1].top) + pr::scale_exp(rb[1].top));
    return pr::scale_exp(ra[0].top) + pr::scale_exp(rb[mat].top);
  }
  __device__ __forceinline__ bool second(int i, int n) const { return P == kForward ? i == 1 : P == kWeights && n >= ld; }
  __device__ __forceinline__ int row(int, int, int) const { return 0; }
  template <int W>
  __device__ __forceinline__ int fetch(int, int, bool) const { return 0; }

  // Forward: a warp's 32 rows of 16 columns of a (sums[0]) and of u (sums[1]).
  template <int MINE>
  __device__ __forceinline__ void finish(int m0, int tile_n, int c, int lane, float* scratch, float (&sums)[MINE][16]) const {
    static_assert(MINE == 2, "the columns of both matrices");
    const int n = tile_n * 64 + c * 16;
    if (n >= N) return;
    const size_t at = (size_t)m0 * N + n;
    if (pre[0]) {
      send(pre[0] + at, m0, n, lane, scratch, sums[0]);
      send(pre[1] + at, m0, n, lane, scratch, sums[1]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) sums[0][j] = gated::act(sums[0][j], act) * sums[1][j];
    send(out[0] + at, m0, n, lane, scratch, sums[0]);
  }
  __device__ __forceinline__ void send(float* dst, int m0, int n, int lane, float* scratch, const float (&v)[16]) const {
    if (vec) tc::block_to_rows<true>(scratch, lane, v, dst, N, M - m0, N - n, accumulate != 0);
    else tc::block_to_rows<false>(scratch, lane, v, dst, N, M - m0, N - n, accumulate != 0);
  }
  // 32 rows from m0 on and 16 columns from n on of the product.
  __device__ __forceinline__ void block(int m0, int n, int lane, float* scratch, const float (&v)[16]) const {
    const int mat = P == kWeights && n >= ld ? 1 : 0, c = n - mat * ld;
    if (c >= N) return;
    send(out[mat] + (size_t)m0 * N + c, m0, c, lane, scratch, v);
  }
  int sum_splits(nrs_ctx* ctx, const tc::SplitInfo& sp) const;
};

// The splits' partial products, four columns a thread, added up in order.  (8 MB of them in 2.5 us where a value a thread,
// its place found by two 64-bit divisions, took 7.)
template <Product P>
__global__ void __launch_bounds__(256) gated_splits_kernel(const GatedPolicy<P> pol, const tc::SplitInfo sp, NrsFastDiv div /*of quads*/) {
  NRS_PDL_PROLOGUE();
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  uint32_t row, q;
  div.divmod(i, row, q);
  if ((int)row >= pol.M) return;
  const int n = 4 * (int)q, mat = P == kWeights && n >= pol.ld ? 1 : 0, c = n - mat * pol.ld;
  const bool whole = sp.n_total % 4 == 0;
  const size_t per = (size_t)sp.rows_total * sp.n_total;
  const float* src = sp.partial + (size_t)row * sp.n_total + n;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int z = 0; z < sp.splits; ++z) {
    const float4 o = tc::load_guarded(src + z * per, sp.n_total - n, whole);
    v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
  }
  if (c >= pol.N) return;
  float* dst = pol.out[mat] + (size_t)row * pol.N + c;
  if (pol.accumulate) {
    const float4 o = tc::load_guarded(dst, pol.N - c, pol.vec);
    v = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
  }
  tc::store_guarded(dst, v, pol.N - c, pol.vec);
}
template <Product P>
int GatedPolicy<P>::sum_splits(nrs_ctx* ctx, const tc::SplitInfo& sp) const {
  const uint32_t quads = (uint32_t)(sp.n_total + 3) / 4;   // (a split product is at most half a wave of tiles)
  NRS_PDL_LAUNCH(gated_splits_kernel<P>, ((uint32_t)M * quads + 255) / 256, 256, 0, ctx->stream, *this, sp, NrsFastDiv((int)quads));
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

// ------------------------------------------------------------------------------------------------ operand planes

// A tensor [rows][cols] on its way to planes, or (a, u given) the two that dh, a and u make, da and du.
struct Job {
  const float* src;
  const float *a, *u;
  __half *hi, *lo;
  NrsRange* range;          // of da and du: two
  const NrsRange *other, *with, *other_with;   // of a weight in dx's sum: the other weight's, and those of what the two are multiplied by
  int rows, cols, pad;      // pad: a row's values in the planes, cols rounded up to 64
  long ld;                  // values between rows of the planes
  unsigned first, blocks;   // of the launch
  NrsFastDiv div;           // of a row's units
  bool vec, whole;          // rows, or the tensor at least, start on 16 bytes
};
struct Jobs {
  Job j[4];
  int count, act;
};

__device__ __forceinline__ void eight(float (&v)[8], const float* p, int left, bool vec) {
  if (vec && left >= 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.0f;
  }
}
__device__ __forceinline__ void put8(__half* hi, __half* lo, size_t at, const float (&v)[8], float scale) {
  uint2 h0, l0, h1, l1;
  pr::split4(make_float4(v[0], v[1], v[2], v[3]), scale, &h0, &l0);
  pr::split4(make_float4(v[4], v[5], v[6], v[7]), scale, &h1, &l1);
  *reinterpret_cast<uint4*>(hi + at) = make_uint4(h0.x, h0.y, h1.x, h1.y);
  *reinterpret_cast<uint4*>(lo + at) = make_uint4(l0.x, l0.y, l1.x, l1.y);
}

__device__ __forceinline__ const Job& job_of(const Jobs& jobs) {
  int which = 0;
  while (which + 1 < jobs.count && blockIdx.x >= jobs.j[which + 1].first) ++which;
  return jobs.j[which];
}

// The largest magnitude of each tensor into its range.  Of da and du themselves, exponentials and all: a bound from dh u and
// dh a is cheaper, but a gate far to the left, which passes nothing on, would set the exponent for all the others.
__global__ void __launch_bounds__(256, 3) gated_measure_kernel(const Jobs jobs) {
  NRS_PDL_PROLOGUE();
  const Job& q = job_of(jobs);
  const size_t count = (size_t)q.rows * q.cols, units = q.whole ? count / 8 : 0, step = (size_t)q.blocks * 256;   // (whole: 16-byte accesses)
  const bool grads = q.a != nullptr;
  uint32_t top = 0, top_u = 0;
  auto see = [&](float (&g)[8], float (&a)[8], float (&u)[8]) {
    if (grads) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f, d;
        gated::act_both(a[i], jobs.act, f, d);
        a[i] = g[i] * u[i] * d;
        u[i] = g[i] * f;
      }
      top = pr::seen_all(top, a);
      top_u = pr::seen_all(top_u, u);
    } else {
      top = pr::seen_all(top, g);
    }
  };
  const size_t me = (size_t)(blockIdx.x - q.first) * 256 + threadIdx.x;
  constexpr int kDeep = 2;
  for (size_t i0 = me; i0 < units; i0 += kDeep * step) {
    float g[kDeep][8], a[kDeep][8], u[kDeep][8];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const size_t at = 8 * min(i0 + k * step, units - 1);   // (past the end: the last one again)
      eight(g[k], q.src + at, 8, true);
      if (grads) {
        eight(a[k], q.a + at, 8, true);
        eight(u[k], q.u + at, 8, true);
      }
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) see(g[k], a[k], u[k]);
  }
  for (size_t i = 8 * units + me; i < count; i += step) {   // what is left of them, or all
    float g[8] = {q.src[i]}, a[8] = {}, u[8] = {};
    if (grads) { a[0] = q.a[i]; u[0] = q.u[i]; }
    see(g, a, u);
  }
  // (one atomic a block: those of ten thousand warps on one word took longer than the pass)
  __shared__ uint32_t tops[2][8];
  top = __reduce_max_sync(0xffffffffu, top);
  top_u = __reduce_max_sync(0xffffffffu, top_u);
  if ((threadIdx.x & 31) == 0) { tops[0][threadIdx.x >> 5] = top; tops[1][threadIdx.x >> 5] = top_u; }
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  if (warp < (grads ? 2 : 1)) pr::report(q.range + warp, (threadIdx.x & 31) < 8 ? tops[warp][threadIdx.x & 31] : 0u);
}

// The pairs, zeros from cols to pad: eight values a thread where rows start on 16 bytes, else 128 values a warp, value by value
// (eight neighbours a thread, loaded one by one, touch eight lines with every load).
__global__ void __launch_bounds__(256, 4) gated_stage_kernel(const Jobs jobs) {
  NRS_PDL_PROLOGUE();
  const Job& q = job_of(jobs);
  const bool grads = q.a != nullptr;
  int e = pr::scale_exp(q.range->top);
  if (q.other) e = min(e, pr::scale_exp(q.other->top) + pr::scale_exp(q.other_with->top) - pr::scale_exp(q.with->top));
  const float scale = e < -126 ? 0.0f : pr::pow2(e), scale_u = grads ? pr::scale_of(q.range[1].top) : 0.0f;   // (0: nothing of it reaches the sum)
  if (q.vec) {
    const uint32_t units = (uint32_t)q.rows * (uint32_t)(q.pad / 8), step = q.blocks * 256;   // (the launcher checks the range)
    for (uint32_t i = (blockIdx.x - q.first) * 256 + threadIdx.x; i < units; i += step) {
      uint32_t row, col;
      q.div.divmod(i, row, col);
      col *= 8;
      const int left = q.cols - (int)col;
      const size_t from = (size_t)row * q.cols + col, at = (size_t)row * q.ld + col;
      float g[8];
      eight(g, q.src + from, left, true);
      if (!grads) {
        put8(q.hi, q.lo, at, g, scale);
        continue;
      }
      float a[8], u[8];
      eight(a, q.a + from, left, true);
      eight(u, q.u + from, left, true);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float f, d;
        gated::act_both(a[k], jobs.act, f, d);
        a[k] = g[k] * u[k] * d;
        u[k] = g[k] * f;
      }
      put8(q.hi, q.lo, at, a, scale);
      put8(q.hi, q.lo, at + q.pad, u, scale_u);
    }
    return;
  }
  const uint32_t units = (uint32_t)q.rows * (uint32_t)((q.pad + 127) / 128), step = q.blocks * 8;
  for (uint32_t i = (blockIdx.x - q.first) * 8 + (threadIdx.x >> 5); i < units; i += step) {
    uint32_t row, seg;
    q.div.divmod(i, row, seg);
    const int c0 = (int)seg * 128 + (threadIdx.x & 31);
    const size_t from = (size_t)row * q.cols + c0, at = (size_t)row * q.ld + c0;
    float g[4], a[4] = {}, u[4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool on = c0 + 32 * k < q.cols;
      g[k] = on ? q.src[from + 32 * k] : 0.0f;
      if (grads) {
        a[k] = on ? q.a[from + 32 * k] : 0.0f;
        u[k] = on ? q.u[from + 32 * k] : 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (c0 + 32 * k >= q.pad) break;
      if (!grads) {
        pr::put(q.hi, q.lo, at + 32 * k, g[k], scale);
        continue;
      }
      float f, d;
      gated::act_both(a[k], jobs.act, f, d);
      pr::put(q.hi, q.lo, at + 32 * k, g[k] * u[k] * d, scale);
      pr::put(q.hi, q.lo, at + q.pad + 32 * k, g[k] * f, scale_u);
    }
  }
}

int round64(int v) { return (v + 63) / 64 * 64; }

struct Planes {
  void *hi, *lo;
  NrsRange* range;          // one for each matrix in a row
  int pad, ld;              // values of one matrix in a row, and of a row
};
int open_planes(nrs_ctx* ctx, int slot, int rows, int cols, int side_by_side, Planes* out) {
  out->pad = round64(cols);
  out->ld = side_by_side * out->pad;
  const int st = nrs_ws_planes(ctx, slot, (size_t)rows * out->ld, true, &out->hi, &out->lo);
  return st == NRS_OK ? nrs_range_renew(ctx, out->hi, &out->range, side_by_side) : st;
}
bool aligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}
void add_job(Jobs* jobs, const float* src, const float* a, const float* u, int rows, int cols, const Planes& to, int mat) {
  Job& q = jobs->j[jobs->count++];
  q.src = src; q.a = a; q.u = u;
  q.hi = (__half*)to.hi + (size_t)mat * to.pad; q.lo = (__half*)to.lo + (size_t)mat * to.pad;
  q.range = to.range + mat;
  q.rows = rows; q.cols = cols; q.pad = to.pad; q.ld = to.ld;
  q.whole = aligned({src, a, u});
  q.vec = q.whole && cols % 4 == 0;
  q.div = NrsFastDiv(q.vec ? to.pad / 8 : (to.pad + 127) / 128);
}
// Blocks by the jobs' bytes, up to eight an SM in all (a job's own units permitting).
int run_jobs(nrs_ctx* ctx, Jobs& jobs) {
  for (int pass = 0; pass < 2; ++pass) {   // measure, then write
    double work[4], all = 0.0;
    for (int i = 0; i < jobs.count; ++i) all += work[i] = (double)jobs.j[i].rows * jobs.j[i].pad * (jobs.j[i].a ? (pass ? 5.0 : 3.0) : (pass ? 2.0 : 1.0));
    unsigned at = 0;
    for (int i = 0; i < jobs.count; ++i) {
      Job& q = jobs.j[i];
      const unsigned most = (unsigned)(((size_t)q.rows * (q.pad / 8) + 255) / 256), share = (unsigned)(work[i] / all * 8 * ctx->sm_count) + 1;
      q.first = at;
      q.blocks = std::min(most, share);
      at += q.blocks;
    }
    if (pass) NRS_PDL_LAUNCH(gated_stage_kernel, at, 256, 0, ctx->stream, jobs);
    else NRS_PDL_LAUNCH(gated_measure_kernel, at, 256, 0, ctx->stream, jobs);
    NRS_LAUNCHED(ctx);
  }
  return NRS_OK;
}

// Planes with K along the rows: [mat][row][cols].
bool map_k(CUtensorMap* t, const void* base, const Planes& p, int cols, int rows, int mats, int box_rows) {
  const uint64_t dim[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)mats}, str[2] = {(uint64_t)p.ld, (uint64_t)p.pad};
  const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
  return tc::encode_tmap(t, base, true, 3, dim, str, box);
}
// Planes with K across the rows: [block of 64 columns][k][64].
bool map_mn(CUtensorMap* t, const void* base, const Planes& p, int k, int box_cols) {
  const uint64_t dim[3] = {64, (uint64_t)k, (uint64_t)(p.ld / 64)}, str[2] = {(uint64_t)p.ld, 64};
  const uint32_t box[3] = {64, 64, (uint32_t)(box_cols / 64)};
  return tc::encode_tmap(t, base, true, 3, dim, str, box, true);
}

// The product of A [rows] and B [cols, padding included]; k: its length (input: of one matrix).
template <int BN, bool PAIR, Product P>
int run(nrs_ctx* ctx, const Planes& A, const Planes& B, GatedPolicy<P> pol, int rows, int cols, int k, int* splits = nullptr) {
  constexpr int kBCols = PAIR || P == kForward ? BN / 2 : BN;   // of B in one load
  CUtensorMap a[2], b[2];
  bool ok = true;
  for (int i = 0; i < 2; ++i) {
    const void *pa = i ? A.lo : A.hi, *pb = i ? B.lo : B.hi;
    ok = ok && (P == kWeights ? map_mn(&a[i], pa, A, k, tc::BM) : map_k(&a[i], pa, A, k, rows, P == kInput ? 2 : 1, tc::BM));
    ok = ok && (P == kInput ? map_k(&b[i], pb, B, k, cols, 2, kBCols) : map_mn(&b[i], pb, B, k, kBCols));
  }
  NRS_REQUIRE(ctx, ok, NRS_ERR_CUDA, "gated layer: cuTensorMapEncodeTiled failed (%d x %d x %d)", rows, cols, k);
  pol.ra = A.range;
  pol.rb = B.range;
  const int kb = P == kInput ? 2 * (A.pad / 64) : (k + 63) / 64;
  return tc::launch<BN, 2, PAIR, 64, GatedPolicy<P>>(ctx, a[0], a[1], b[0], b[1], pol, (rows + tc::BM - 1) / tc::BM, cols, 1, kb,
                                                     tc::Ranges{}, nullptr, nullptr, splits);
}

bool applies(const nrs_ctx* ctx, const Shape& s) {
  // (from 16 rows on, as the ungated products; the staging passes count eights in 32 bits)
  if (s.n > (1 << 24) || s.k > (1 << 24)) return false;
  const uint64_t m = s.m, n = round64(s.n), k = round64(s.k), most = 1ull << 33;
  return ctx->math_mode == NRS_MATH_3XTF32 && tc::tensor_map_encoder() && s.m >= 16 && s.n >= 32 && s.k >= 32 && m * n <= most && m * k <= most && k * n <= most;
}

}  // namespace

int nrs_tc_gated_fwd(nrs_ctx* ctx, const Shape& s, const float* x, const float* w_gate, const float* w_up, float* h, float* pre_gate, float* pre_up) {
  if (!applies(ctx, s)) return NRS_ERR_UNSUPPORTED;
  Planes X{}, W{};
  int st = open_planes(ctx, NRS_WS_A, s.m, s.k, 1, &X);
  if (st == NRS_OK) st = open_planes(ctx, NRS_WS_B, s.k, s.n, 2, &W);
  if (st != NRS_OK) return st;
  Jobs jobs{};
  add_job(&jobs, x, nullptr, nullptr, s.m, s.k, X, 0);
  add_job(&jobs, w_gate, nullptr, nullptr, s.k, s.n, W, 0);
  add_job(&jobs, w_up, nullptr, nullptr, s.k, s.n, W, 1);
  st = run_jobs(ctx, jobs);
  if (st != NRS_OK) return st;
  GatedPolicy<kForward> pol{};
  pol.out[0] = h; pol.pre[0] = pre_gate; pol.pre[1] = pre_up;
  pol.M = s.m; pol.N = s.n; pol.ld = W.pad; pol.act = s.act;
  pol.vec = s.n % 4 == 0 && aligned({h, pre_gate, pre_up});
  NrsProfScope prof(ctx, NRS_PROF_GEMM, 4.0 * s.m * s.n * s.k);
  // Pairs take 395 clocks per 32 values of K a round of 74, single tiles 530 a round of 148 (plan_tile's table).
  const long tm = (s.m + 127) / 128, tn = W.pad / 64, sms = ctx->sm_count;
  const long pairs = ((tm + 1) / 2 * tn + sms / 2 - 1) / (sms / 2) * 395, singles = (tm * tn + sms - 1) / sms * 530;
  return pairs <= singles ? run<128, true, kForward>(ctx, X, W, pol, s.m, W.ld, s.k) : run<128, false, kForward>(ctx, X, W, pol, s.m, W.ld, s.k);
}

int nrs_tc_gated_bwd(nrs_ctx* ctx, const Shape& s, const float* x, const float* w_gate, const float* w_up, const float* pre_gate, const float* pre_up,
                     const float* dh, float* dx, float* dw_gate, float* dw_up, int acc_x, int acc_w) {
  if (!applies(ctx, s)) return NRS_ERR_UNSUPPORTED;
  Planes D{}, X{}, W{};
  int st = open_planes(ctx, NRS_WS_GATED, s.m, s.n, 2, &D);
  if (st == NRS_OK && dw_gate) st = open_planes(ctx, NRS_WS_A, s.m, s.k, 1, &X);
  if (st == NRS_OK && dx) st = open_planes(ctx, NRS_WS_B, s.k, s.n, 2, &W);
  if (st != NRS_OK) return st;
  Jobs jobs{};
  jobs.act = s.act;
  add_job(&jobs, dh, pre_gate, pre_up, s.m, s.n, D, 0);
  if (dw_gate) add_job(&jobs, x, nullptr, nullptr, s.m, s.k, X, 0);
  if (dx) {
    add_job(&jobs, w_gate, nullptr, nullptr, s.k, s.n, W, 0);
    add_job(&jobs, w_up, nullptr, nullptr, s.k, s.n, W, 1);
    for (int mat = 0; mat < 2; ++mat) {
      Job& q = jobs.j[jobs.count - 2 + mat];
      q.other = W.range + 1 - mat; q.with = D.range + mat; q.other_with = D.range + 1 - mat;
    }
  }
  st = run_jobs(ctx, jobs);
  if (st != NRS_OK) return st;
  int splits = 0;   // of the product for dx (0: there is none)
  if (dx) {
    GatedPolicy<kInput> pol{};
    pol.out[0] = dx; pol.M = s.m; pol.N = s.k; pol.ld = D.pad; pol.accumulate = acc_x;
    pol.vec = s.k % 4 == 0 && aligned({dx});
    NrsProfScope prof(ctx, NRS_PROF_GEMM, 4.0 * s.m * s.n * s.k);
    const tc::TilePlan t = tc::plan_tile(ctx, (s.m + 127) / 128, s.k, 1, D.ld / 32, true, 0.004, false, false);
#define NRS_RUN(BN_, PAIR_) run<BN_, PAIR_, kInput>(ctx, D, W, pol, s.m, s.k, s.n, &splits)
    st = t.bn == 128 ? (t.pair ? NRS_RUN(128, true) : NRS_RUN(128, false)) : (t.pair ? NRS_RUN(64, true) : NRS_RUN(64, false));
#undef NRS_RUN
    if (st != NRS_OK) return st;
  }
  if (dw_gate) {
    GatedPolicy<kWeights> pol{};
    pol.out[0] = dw_gate; pol.out[1] = dw_up; pol.M = s.k; pol.N = s.n; pol.ld = D.pad; pol.accumulate = acc_w;
    pol.vec = s.n % 4 == 0 && aligned({dw_gate, dw_up});
    // It reads nothing that the product for dx wrote, and starts on the SMs that one leaves idle; but not over partial sums
    // that are still being added up.
    pol.independent = splits == 1;
    NrsProfScope prof(ctx, NRS_PROF_GEMM, 4.0 * s.m * s.n * s.k);
    const tc::TilePlan t = tc::plan_tile(ctx, (s.k + 127) / 128, D.ld, 1, (s.m + 31) / 32, true, 0.004, false, false);
#define NRS_RUN(BN_, PAIR_) run<BN_, PAIR_, kWeights>(ctx, X, D, pol, s.k, D.ld, s.m)
    // (columns of 64 in a CTA's share of B: no pair of 64)
    st = t.bn == 128 && t.pair ? NRS_RUN(128, true) : t.bn == 128 ? NRS_RUN(128, false) : NRS_RUN(64, false);
#undef NRS_RUN
  }
  return st;
}
