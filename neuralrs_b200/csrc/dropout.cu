// Dropout and spatial dropout: the mask multiply of the reference (mask_mul, src/cuda/nn/dropout.rs:17-22;
// mask_mul_channels, src/cuda/nn/dropout2d.rs:18-27) and a device-side mask generator.
//
// The reference draws the mask on the host with the thread-local generator of the `rand` crate and uploads it
// (dropout.rs:45-48): a value per element, 0 with probability p, else 1/(1-p).  Uploading a mask per layer per
// step would put the host on the training path, so the mask is made on the device from a counter-based
// generator (Philox-4x32-10, Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC'11): element i of
// a call is word i%4 of the block at counter (offset + i/4) under the context's 64-bit seed, u = (word >> 8) *
// 2^-24 in [0,1), mask = u < p ? 0 : 1/(1-p).  The same seed and offset give the same mask on any launch
// shape; a caller that wants the reference's own masks passes them to nrs_mask_mul instead.
#include <cmath>

#include "igemm_problems.cuh"
#include "nrs_internal.h"
#include "philox.cuh"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float mask_value(uint32_t word, float p, float scale) {
  return nrs_rng::uniform01(word) < p ? 0.0f : scale;
}

__global__ void __launch_bounds__(kThreads)
dropout_mask_kernel(float* __restrict__ mask, size_t count, float p, float scale, uint64_t seed, uint64_t offset) {
  NRS_PDL_PROLOGUE();
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  const size_t blocks = (count + 3) / 4;
  const bool vec = (reinterpret_cast<uintptr_t>(mask) & 15) == 0;
  for (size_t b = (size_t)blockIdx.x * blockDim.x + threadIdx.x; b < blocks; b += stride) {
    uint32_t ctr[4];
    nrs_rng::block(seed, offset + b, ctr);
    const float4 v = make_float4(mask_value(ctr[0], p, scale), mask_value(ctr[1], p, scale),
                                 mask_value(ctr[2], p, scale), mask_value(ctr[3], p, scale));
    const size_t i = b * 4;
    if (vec && i + 4 <= count) {
      reinterpret_cast<float4*>(mask)[b] = v;
    } else {
      const float e[4] = {v.x, v.y, v.z, v.w};
      for (int j = 0; j < 4 && i + j < count; ++j) mask[i + j] = e[j];
    }
  }
}

// out (+)= a * mask[i / hw]; hw == 1 is the per-element mask.
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
mask_mul_kernel(const float* __restrict__ a, const float* __restrict__ mask, float* out, size_t total, int hw,
                int accumulate) {
  NRS_PDL_PROLOGUE();
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  const size_t tid = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (VEC) {   // hw == 1 (a mask vector per data vector) or hw % 4 == 0 (one mask value per data vector)
    for (size_t i = tid; i < total / 4; i += stride) {
      const float4 v = reinterpret_cast<const float4*>(a)[i];
      float4 m;
      if (hw == 1) {
        m = reinterpret_cast<const float4*>(mask)[i];
      } else {
        const float s = mask[i * 4 / hw];
        m = make_float4(s, s, s, s);
      }
      float4 r = make_float4(v.x * m.x, v.y * m.y, v.z * m.z, v.w * m.w);
      float4* dst = reinterpret_cast<float4*>(out) + i;
      if (accumulate) {
        const float4 o = *dst;
        r = make_float4(o.x + r.x, o.y + r.y, o.z + r.z, o.w + r.w);
      }
      *dst = r;
    }
    if (tid < (total & 3)) {   // tail of a per-element mask whose length is not a multiple of four
      const size_t i = (total & ~(size_t)3) + tid;
      const float r = a[i] * mask[i / hw];
      out[i] = accumulate ? out[i] + r : r;
    }
  } else {
    for (size_t i = tid; i < total; i += stride) {
      const float r = a[i] * mask[i / hw];
      out[i] = accumulate ? out[i] + r : r;
    }
  }
}

// Dropout without a mask in memory: out = a * m (+ residual), or out (+)= a * m, with the mask of dropout_mask_kernel made
// again wherever it is needed.  What a stored mask costs, 4 bytes written and read again in both passes and kept between
// them, is spent on twenty wide multiplications per block of four instead, which run under the loads.
// u < p is asked of the word itself: u = (word >> 8) 2^-24, so it holds for words up to 2^8 ceil(2^24 p) - 1 (p = 0, where
// none are, has a dropped value's factor 1 instead).
// Bound by memory, with the generator close behind: it takes half of the issue slots at full memory rate.  67 M values, both
// passes: 205 us with u made and compared as a float, 199 as an integer, 190 compared as it comes and with counters whose
// upper half all threads of a launch share (a call that crosses 2^32 takes two launches), which spares two of twenty
// products, 178 with the form without a second operand compiled apart (39 registers, six blocks an SM); 165 with a toy
// generator in its place.  The copy rate allows 166.
struct Draw {
  uint64_t seed, first;
  uint32_t last;           // words up to here are dropped ones
  float dropped, kept;     // their factor, and the others'
  __device__ __forceinline__ float factor(uint32_t word) const { return word <= last ? dropped : kept; }
};
constexpr int kUnroll = 4;   // vectors of a thread under way together

// Four elements from 4 * b on, of `total`; VEC: 16-byte accesses to all that are whole.
template <bool VEC>
__device__ __forceinline__ float4 load_four(const float* a, size_t b, size_t total) {
  if (VEC && 4 * b + 4 <= total) return reinterpret_cast<const float4*>(a)[b];
  float e[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (4 * b + j < total) e[j] = a[4 * b + j];
  return make_float4(e[0], e[1], e[2], e[3]);
}
template <bool VEC>
__device__ __forceinline__ void store_four(float* out, size_t b, size_t total, float4 y) {
  if (VEC && 4 * b + 4 <= total) {
    reinterpret_cast<float4*>(out)[b] = y;
  } else {
    const float e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * b + j < total) out[4 * b + j] = e[j];
  }
}

// A value per element: a block's four words serve four neighbouring elements.
template <bool VEC, bool ADD>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const float* a, const float* residual, float* out, size_t total, const Draw draw, int accumulate) {
  NRS_PDL_PROLOGUE();
  const size_t groups = (total + 3) / 4;
  const float* add = ADD ? (accumulate ? out : residual) : nullptr;
  for (size_t base = (size_t)blockIdx.x * (kThreads * kUnroll) + threadIdx.x; base < groups; base += (size_t)gridDim.x * (kThreads * kUnroll)) {
    float4 v[kUnroll], r[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const size_t b = base + (size_t)u * kThreads;
      v[u] = r[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (b >= groups) continue;
      v[u] = load_four<VEC>(a, b, total);
      if (ADD) r[u] = load_four<VEC>(add, b, total);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const size_t b = base + (size_t)u * kThreads;
      if (b >= groups) continue;
      uint32_t w[4];
      nrs_rng::block(draw.seed, (draw.first >> 32 << 32) | (uint32_t)((uint32_t)draw.first + (uint32_t)b), w);
      const float4 m = make_float4(draw.factor(w[0]), draw.factor(w[1]), draw.factor(w[2]), draw.factor(w[3]));
      float4 y = make_float4(v[u].x * m.x, v[u].y * m.y, v[u].z * m.z, v[u].w * m.w);
      if (ADD) {   // rounded once, as mask_mul_kernel does (but for the rest of a length that is no multiple of four)
        if (VEC && 4 * b + 4 > total) y = make_float4(__fadd_rn(r[u].x, y.x), __fadd_rn(r[u].y, y.y), __fadd_rn(r[u].z, y.z), 0.0f);
        else y = make_float4(fmaf(v[u].x, m.x, r[u].x), fmaf(v[u].y, m.y, r[u].y), fmaf(v[u].z, m.z, r[u].z), fmaf(v[u].w, m.w, r[u].w));
      }
      store_four<VEC>(out, b, total, y);
    }
  }
}

// A value per plane of hw > 1 elements.  Four planes have one counter block and are hw whole vectors of four, whatever hw is; a
// vector meets two of them at most.  A block of threads takes a stretch of vectors, loads it, draws the counter blocks that it
// meets, one a thread, into shared memory, and multiplies.  [256][512][7][7], both passes: 26 us, with a counter block for every
// element 69, with a stored mask 40; [256][64][32][32] 48, 58 and 60 (floors 16 and 42).
template <bool VEC, bool ADD>
__global__ void __launch_bounds__(kThreads)
dropout_planes_kernel(const float* a, const float* residual, float* out, size_t total, uint32_t hw, NrsFastDiv by_hw, const Draw draw, int accumulate) {
  NRS_PDL_PROLOGUE();
  constexpr uint32_t kStretch = kThreads * kUnroll;
  __shared__ uint8_t s_kept[2][kStretch / 2 + 2];   // of every four planes met (at most one for two vectors, and a broken one): a bit for each
  const size_t vectors = (total + 3) / 4;
  const float* add = ADD ? (accumulate ? out : residual) : nullptr;
  int turn = 0;                                     // (two stretches' bits: the one before may still be read)
  for (size_t base = (size_t)blockIdx.x * kStretch; base < vectors; base += (size_t)gridDim.x * kStretch, turn ^= 1) {
    float4 v[kUnroll], r[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const size_t b = base + u * kThreads + threadIdx.x;
      v[u] = r[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (b >= vectors) continue;
      v[u] = load_four<VEC>(a, b, total);
      if (ADD) r[u] = load_four<VEC>(add, b, total);
    }
    const size_t four0 = base >> 32 ? base / hw : (size_t)((uint32_t)base / hw);       // the four planes that the stretch starts in
    const uint32_t at0 = (uint32_t)(base - four0 * hw);                                // and its first vector there
    const uint32_t count = (uint32_t)min((size_t)kStretch, vectors - base);
    auto four_of = [&](uint32_t at) { return hw >= kStretch ? (at >= hw ? 1u : 0u) : by_hw.div(at); };
    const uint32_t fours = four_of(at0 + count - 1) + 1;
    for (uint32_t i = threadIdx.x; i < fours; i += kThreads) {
      uint32_t w[4];
      nrs_rng::block(draw.seed, draw.first + four0 + i, w);
      s_kept[turn][i] = (uint8_t)((w[0] > draw.last) | (w[1] > draw.last) << 1 | (w[2] > draw.last) << 2 | (w[3] > draw.last) << 3);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t i = u * kThreads + threadIdx.x;
      if (i >= count) continue;
      const uint32_t at = at0 + i, four = four_of(at);
      const uint64_t e = 4ull * (at - four * hw);                                      // the vector's first element among the four planes'
      const uint32_t plane = (e >= hw) + (e >= 2ull * hw) + (e >= 3ull * hw), left = (uint32_t)min(4ull, (unsigned long long)((plane + 1ull) * hw - e));
      const uint32_t kept = s_kept[turn][four] >> plane;
      const float f = kept & 1 ? draw.kept : draw.dropped, g = kept & 2 ? draw.kept : draw.dropped;   // (left: elements of the first)
      const float4 m = make_float4(f, left > 1 ? f : g, left > 2 ? f : g, left > 3 ? f : g);
      float4 y = make_float4(v[u].x * m.x, v[u].y * m.y, v[u].z * m.z, v[u].w * m.w);
      if (ADD) y = make_float4(fmaf(v[u].x, m.x, r[u].x), fmaf(v[u].y, m.y, r[u].y), fmaf(v[u].z, m.z, r[u].z), fmaf(v[u].w, m.w, r[u].w));
      store_four<VEC>(out, base + i, total, y);
    }
  }
}

unsigned ew_blocks(const nrs_ctx* ctx, size_t work_items) {
  const size_t want = (work_items + kThreads - 1) / kThreads;
  const size_t cap = (size_t)ctx->sm_count * 16;
  return (unsigned)(want < 1 ? 1 : (want > cap ? cap : want));
}

}  // namespace

int nrs_rng_seed(nrs_ctx* ctx, uint64_t seed) {
  NRS_REQUIRE_CTX(ctx);
  ctx->rng_seed = seed;
  ctx->rng_offset = 0;
  return NRS_OK;
}

int nrs_rng_offset(nrs_ctx* ctx, uint64_t* offset) {
  NRS_REQUIRE_CTX(ctx);
  NRS_REQUIRE(ctx, offset, NRS_ERR_ARG, "nrs_rng_offset: null output");
  *offset = ctx->rng_offset;
  return NRS_OK;
}

int nrs_dropout_mask(nrs_ctx* ctx, float* mask, size_t count, float p) {
  NRS_REQUIRE_CTX(ctx);
  NRS_REQUIRE(ctx, p >= 0.0f && p <= 1.0f, NRS_ERR_ARG, "nrs_dropout_mask: probability %g outside [0,1]", (double)p);
  if (count == 0) return NRS_OK;
  NRS_REQUIRE(ctx, mask, NRS_ERR_ARG, "nrs_dropout_mask: null mask");
  const size_t blocks = (count + 3) / 4;
  // p == 1 drops everything (u < 1 always holds), so the infinite scale is never used: the reference's
  // 1/(1-p) is kept as it is (dropout.rs:38).
  const float scale = 1.0f / (1.0f - p);
  uint64_t first = 0, advance = 0;
  nrs_rng_window(ctx, count, &first, &advance);   // a data-parallel shard draws its samples' part of the global mask
  NRS_PDL_LAUNCH(dropout_mask_kernel, ew_blocks(ctx, blocks), kThreads, 0, ctx->stream, mask, count, p, scale, ctx->rng_seed,
                 first);
  NRS_LAUNCHED(ctx);
  ctx->rng_offset += advance;
  return NRS_OK;
}

int nrs_mask_mul(nrs_ctx* ctx, const float* a, const float* mask, float* out, size_t total, int hw, int accumulate) {
  NRS_REQUIRE_CTX(ctx);
  NRS_REQUIRE(ctx, hw >= 1, NRS_ERR_SHAPE, "nrs_mask_mul: bad plane size %d", hw);
  if (total == 0) return NRS_OK;
  NRS_REQUIRE(ctx, a && mask && out, NRS_ERR_ARG, "nrs_mask_mul: null tensor");
  NRS_REQUIRE(ctx, total % (size_t)hw == 0, NRS_ERR_SHAPE, "nrs_mask_mul: %zu elements are not whole planes of %d", total, hw);
  const bool al = (((uintptr_t)a | (uintptr_t)out) & 15) == 0;
  const bool vec = al && ((hw == 1 && ((uintptr_t)mask & 15) == 0) || (hw & 3) == 0);
  if (vec) {
    NRS_PDL_LAUNCH(mask_mul_kernel<true>, ew_blocks(ctx, total / 4 + 1), kThreads, 0, ctx->stream, a, mask, out, total, hw, accumulate);
  } else {
    NRS_PDL_LAUNCH(mask_mul_kernel<false>, ew_blocks(ctx, total), kThreads, 0, ctx->stream, a, mask, out, total, hw, accumulate);
  }
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

int nrs_rng_take(nrs_ctx* ctx, size_t count, uint64_t* seed, uint64_t* first_block) {
  NRS_REQUIRE_CTX(ctx);
  NRS_REQUIRE(ctx, seed && first_block, NRS_ERR_ARG, "nrs_rng_take: null output");
  uint64_t advance = 0;
  *seed = ctx->rng_seed;
  nrs_rng_window(ctx, count, first_block, &advance);   // a data-parallel shard takes its samples' part of the global draw
  ctx->rng_offset += advance;
  return NRS_OK;
}

static int dropout_pass(nrs_ctx* ctx, const char* who, const float* a, const float* residual, float* out, size_t total, int hw, float p,
                        uint64_t seed, uint64_t first, int accumulate) {
  NRS_REQUIRE(ctx, p >= 0.0f && p <= 1.0f, NRS_ERR_ARG, "%s: probability %g outside [0,1]", who, (double)p);
  NRS_REQUIRE(ctx, hw >= 1, NRS_ERR_SHAPE, "%s: bad plane size %d", who, hw);
  if (total == 0) return NRS_OK;
  NRS_REQUIRE(ctx, a && out, NRS_ERR_ARG, "%s: null tensor", who);
  NRS_REQUIRE(ctx, total % (size_t)hw == 0, NRS_ERR_SHAPE, "%s: %zu elements are not whole planes of %d", who, total, hw);
  NrsDeviceGuard on(ctx);
  const uint32_t below = (uint32_t)std::ceil(p * 16777216.0f);
  Draw draw{seed, first, (below << 8) - 1u, 0.0f, 1.0f / (1.0f - p)};   // (p == 1: every word, and the infinite factor is never used)
  if (below == 0) { draw.last = 0; draw.dropped = 1.0f; }
  const bool aligned = (((uintptr_t)a | (uintptr_t)out | (uintptr_t)residual) & 15) == 0;
  while (total > 0) {
    size_t part = total;
    if (hw == 1) {   // up to where the counter's upper half changes
      const uint64_t left = ((uint64_t)1 << 32) - (uint32_t)draw.first;
      if ((total + 3) / 4 > left) part = (size_t)left * 4;
    }
    const size_t want = ((part + 3) / 4 + 4 * kThreads - 1) / (4 * kThreads), cap = (size_t)ctx->sm_count * 16;
    const unsigned blocks = (unsigned)(want > cap ? cap : want);
    const bool add = accumulate || residual;
#define NRS_DROPOUT(VEC_, ADD_)                                                                                                                       \
  if (hw == 1)                                                                                                                                        \
    NRS_PDL_LAUNCH((dropout_kernel<VEC_, ADD_>), blocks, kThreads, 0, ctx->stream, a, residual, out, part, draw, accumulate);                         \
  else                                                                                                                                                \
    NRS_PDL_LAUNCH((dropout_planes_kernel<VEC_, ADD_>), blocks, kThreads, 0, ctx->stream, a, residual, out, part, (uint32_t)hw, NrsFastDiv(hw), draw, accumulate)
    if (aligned && add) {
      NRS_DROPOUT(true, true);
    } else if (aligned) {
      NRS_DROPOUT(true, false);
    } else if (add) {
      NRS_DROPOUT(false, true);
    } else {
      NRS_DROPOUT(false, false);
    }
#undef NRS_DROPOUT
    NRS_LAUNCHED(ctx);
    total -= part;
    draw.first += part / 4;   // (with a total left, a part is whole blocks)
    a += part;
    out += part;
    if (residual) residual += part;
  }
  return NRS_OK;
}

int nrs_dropout_fwd(nrs_ctx* ctx, const float* x, const float* residual, float* y, size_t total, int hw, float p, uint64_t seed,
                    uint64_t first_block) {
  NRS_REQUIRE_CTX(ctx);
  return dropout_pass(ctx, __func__, x, residual, y, total, hw, p, seed, first_block, 0);
}

int nrs_dropout_bwd(nrs_ctx* ctx, const float* g, float* dx, size_t total, int hw, float p, uint64_t seed, uint64_t first_block, int accumulate) {
  NRS_REQUIRE_CTX(ctx);
  return dropout_pass(ctx, __func__, g, nullptr, dx, total, hw, p, seed, first_block, accumulate != 0);
}
