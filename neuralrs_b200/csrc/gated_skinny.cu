// A gated layer's forward pass for some dozen rows (a batch of growing sequences), on the tensor cores without a pass over the
// weights ahead of the product: what bounds it is the weights' way from memory, 8 k n bytes, once.
//
// The product is turned around: 64 columns of Wg and the same 64 of Wu are the 128 rows of an M = 128 UMMA, the rows of x its
// N columns (16 to 128), h^T = W^T x^T.  TMA brings the f32 values as they lie, [k][n] is an MN-major operand already.
// Precision: 3xTF32 with the split made on the way.  The tensor core reads an f32 value cut to 11 bits; eight warps write what
// that leaves, v - cut(v), to a second slot of the same layout, whatever the layout is, and
//   hi.[x_hi ; x_lo] and lo.x_hi
// are issued from the two (kind::tf32, no exponents to measure).  Each slice of 32 values of k leaves tensor memory for f32
// sums in the registers of eight other warps, so the error is that of f32 (chains of 64 erred twice as much).
//
// Work is cut into K-slices of 32 over all column tiles, in a row, and every SM takes an equal stretch (86 tiles of 5504
// columns on 148 SMs would idle two in five): a stretch's share of a tile goes to scratch, and a second launch adds the shares
// up in order, applies the activation and multiplies.
//
// 2048 -> 5504, 90 MB of weights (floor 14 us): 16 rows 25 us, 64 rows 34 us; with one group of splitting warps, which then also
// drained, 31 and 41 us; measuring and staging the weights first 78 us.  A slice costs shared memory 16 KB in, 16 KB out and in
// again for the split, and 32 KB for the UMMAs' reads, about 730 clocks by count, and memory brings one in 710 when all SMs
// ask.  Taken from 2048 and 8192 values of k it costs 0.43 us at 16 rows (some 800 clocks), 0.62 at 64 and 1.0 at 128, where
// x's slice, as large as the weights', is split too and leaves the ring three slots.  An SM has 37 of them here; what is left,
// 9, 10 and 15 us, is two launches: the first one's start and the filling of its ring, the shares and their sum.
#include <algorithm>

#include "gated.h"
#include "tc_common.cuh"

namespace {

using gated::Shape;

constexpr int kSlice = 32;                         // values of k
constexpr int kWBytes = 128 * kSlice * 4;          // a slice of both weights
constexpr int kGroups = 2, kGroupWarps = 4;        // splitting warps: the groups take turns, a slice each, to hide each other's latency
constexpr int kDrainers = 8;                       // warps that drain the accumulators
constexpr int kThreads = 64 + 32 * (kGroups * kGroupWarps + kDrainers);

template <int N>
struct Layout {
  static constexpr int kX = N * kSlice * 4, kSlot = kWBytes + 2 * kX;        // [W][x][x's rest]
  static constexpr int kLo = N == 128 ? 3 : 4;                               // slots of the weights' rest
  static constexpr int kSlots = (200 * 1024 - kLo * kWBytes) / kSlot > 6 ? 6 : (200 * 1024 - kLo * kWBytes) / kSlot;
  static constexpr int kBytes = kSlots * kSlot + kLo * kWBytes + 1024 /*align*/ + 256 /*barriers*/;
  static constexpr int kAcc = 2 * N, kTmem = 2 * kAcc < 32 ? 32 : 2 * kAcc;  // hi.hi | cross, twice
  static constexpr int kCols = N >= 32 ? N / 2 : 16;                         // of a draining warp (16: of half of them)
  static_assert(kSlots >= 3 && kBytes <= 227 * 1024 && kTmem <= 512, "shared memory, tensor memory");
};

struct Work {
  long total;            // slices of all tiles
  int per_tile, slots_max;   // slices of a tile; shares of a tile at most
  float* partial;        // [tile][share][N][128]
  __host__ __device__ long first_of(long cta, long ctas) const { return total * cta / ctas; }
  // The CTA that has slice i.
  __host__ __device__ long owner(long i, long ctas) const {
    long c = i * ctas / total;
    while (c + 1 < ctas && first_of(c + 1, ctas) <= i) ++c;
    while (c > 0 && first_of(c, ctas) > i) --c;
    return c;
  }
};

__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1) { tc::tma_load_2d(dst, m, bar, c0, c1); }

// What the tensor core leaves of four values, rounded to what it reads (cut there, it would lean to zero).
__device__ __forceinline__ float4 rest(float4 v) {
  auto r = [](float x) { return tc::tf32_rn(x - __uint_as_float(__float_as_uint(x) & 0xffffe000u)); };
  return make_float4(r(v.x), r(v.y), r(v.z), r(v.w));
}

template <int N>
__global__ void __launch_bounds__(kThreads, 1)
gated_skinny_kernel(const __grid_constant__ CUtensorMap tm_g, const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ CUtensorMap tm_x, const Work wk,
                    int* __restrict__ err_flag) {
  using L = Layout<N>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* lo_ring = smem + L::kSlots * L::kSlot;
  uint64_t* full = reinterpret_cast<uint64_t*>(lo_ring + L::kLo * kWBytes);
  uint64_t *ready = full + L::kSlots, *empty = ready + L::kSlots, *lo_empty = empty + L::kSlots, *acc_full = lo_empty + L::kLo, *acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const int warp = (int)tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    tc::prefetch_tmap(&tm_g); tc::prefetch_tmap(&tm_u); tc::prefetch_tmap(&tm_x);
    for (int s = 0; s < L::kSlots; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&ready[s], kGroupWarps); tc::mbar_init(&empty[s], 1); }
    for (int s = 0; s < L::kLo; ++s) tc::mbar_init(&lo_empty[s], 1);
    for (int b = 0; b < 2; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], kDrainers); }
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, L::kTmem);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tmem = tc::uniform(*tmem_slot);
  NRS_PDL_WAIT();
  NRS_PDL_TRIGGER();
  const long begin = wk.first_of(blockIdx.x, gridDim.x), end = wk.first_of(blockIdx.x + 1, gridDim.x);

  if (warp == 0) {
    // ---------------- TMA producer
    uint32_t s = 0, ph = 0, issued = 0;
    bool ok = true;
    const int tile0 = (int)(begin / wk.per_tile);   // (stepped along from here: a 64-bit division takes longer than a load's issue)
    int at = (int)(begin - (long)tile0 * wk.per_tile), n0 = tile0 * 64;
    for (long i = begin; i < end; ++i) {
      const int k0 = at * kSlice;
      if (!tc::mbar_wait_warp(&empty[s], ph ^ 1u)) { ok = false; break; }
      if (tc::elect_one()) {
        uint8_t* dst = smem + s * L::kSlot;
        tc::mbar_expect_tx(&full[s], kWBytes + L::kX);
        tma_load(dst, &tm_g, &full[s], n0, k0);
        tma_load(dst + kWBytes / 4, &tm_g, &full[s], n0 + 32, k0);
        tma_load(dst + kWBytes / 2, &tm_u, &full[s], n0, k0);
        tma_load(dst + 3 * kWBytes / 4, &tm_u, &full[s], n0 + 32, k0);
        tma_load(dst + kWBytes, &tm_x, &full[s], k0, 0);
      }
      __syncwarp();
      ++issued;
      if (++s == (uint32_t)L::kSlots) { s = 0; ph ^= 1u; }
      if (++at == wk.per_tile) {
        at = 0;
        n0 += 64;
      }
    }
    if (!ok) {   // loads under way still land here: wait for them, bounded
      if (lane == 0) atomicExch(err_flag, tc::kErrProducerWait);
      for (uint32_t j = issued > (uint32_t)L::kSlots ? issued - L::kSlots : 0; j < issued; ++j)
        if (!tc::mbar_wait_warp(&full[j % L::kSlots], (j / L::kSlots) & 1u)) {
          if (lane == 0) atomicExch(err_flag, tc::kErrDrainWait);
          break;
        }
    }
  } else if (warp == 1) {
    // ---------------- UMMA issuer
    constexpr uint32_t idesc_wide = tc::make_idesc_tf32(128, 2 * N, true, false), idesc = tc::make_idesc_tf32(128, N, true, false);
    uint32_t s = 0, ph = 0, l = 0, buf = 0, aph = 0;
    bool ok = true;
    for (long i = begin; i < end; ++i) {
      if (!tc::mbar_wait_warp(&acc_empty[buf], aph ^ 1u) || !tc::mbar_wait_warp(&ready[s], ph)) { ok = false; break; }
      tc::tc_fence_after_sync();
      const uint32_t d = tmem + buf * (uint32_t)L::kAcc;
      if (tc::elect_one()) {
        const uint32_t w = tc::smem_u32(smem + s * L::kSlot), x = w + kWBytes, wl = tc::smem_u32(lo_ring + l * kWBytes);
#pragma unroll
        for (int k = 0; k < kSlice / 8; ++k) {
          const uint64_t dx = tc::make_smem_desc_sw128(x + k * 32u, 16, 1024);
          tc::umma_tf32(d, tc::make_smem_desc_sw128_32b(w + k * 1024u, kSlice * 128, 512), dx, idesc_wide, k != 0);
          tc::umma_tf32(d + N, tc::make_smem_desc_sw128_32b(wl + k * 1024u, kSlice * 128, 512), dx, idesc, 1);
        }
        tc::umma_commit(&empty[s]);
        tc::umma_commit(&lo_empty[l]);
        tc::umma_commit(&acc_full[buf]);
      }
      __syncwarp();
      if (++s == (uint32_t)L::kSlots) { s = 0; ph ^= 1u; }
      if (++l == (uint32_t)L::kLo) l = 0;
      buf ^= 1u;
      aph ^= buf == 0;
    }
    if (!ok && lane == 0) atomicExch(err_flag, tc::kErrMmaWait);
  } else if (warp < 2 + kGroups * kGroupWarps) {
    // ---------------- split
    const int group = (warp - 2) / kGroupWarps, t = threadIdx.x - 64 - group * 32 * kGroupWarps;
    const uint32_t n = (uint32_t)(end - begin);
    for (uint32_t i = group; i < n; i += kGroups) {
      const uint32_t s = i % L::kSlots, ph = (i / L::kSlots) & 1u, l = i % L::kLo, lph = (i / L::kLo) & 1u;
      if (!tc::mbar_wait_warp(&full[s], ph) || !tc::mbar_wait_warp(&lo_empty[l], lph ^ 1u)) {
        if (lane == 0) atomicExch(err_flag, tc::kErrEpilogueWait);
        break;
      }
      uint8_t* slot = smem + s * L::kSlot;
      const float4* w = reinterpret_cast<const float4*>(slot);
      float4* wl = reinterpret_cast<float4*>(lo_ring + l * kWBytes);
      constexpr int kT = 32 * kGroupWarps, kEach = kWBytes / 16 / kT, kEachX = (L::kX / 16 + kT - 1) / kT;
      float4 v[kEach], y[kEachX];
#pragma unroll
      for (int c = 0; c < kEach; ++c) v[c] = w[c * kT + t];
#pragma unroll
      for (int c = 0; c < kEachX; ++c)
        if (c * kT + t < L::kX / 16) y[c] = w[kWBytes / 16 + c * kT + t];
#pragma unroll
      for (int c = 0; c < kEach; ++c) wl[c * kT + t] = rest(v[c]);
#pragma unroll
      for (int c = 0; c < kEachX; ++c)
        if (c * kT + t < L::kX / 16) reinterpret_cast<float4*>(slot + kWBytes + L::kX)[c * kT + t] = rest(y[c]);
      tc::fence_proxy_async();   // the UMMAs read them
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ready[s]);
    }
  } else {
    // ---------------- drain: the sums of 32 of the tile's rows (TMEM lanes 32 (warp % 4) on) and kCols of x's rows
    const int q = warp & 3, half = (warp - 2 - kGroups * kGroupWarps) >> 2;
    const bool drains = half * L::kCols < N;
    float sums[L::kCols];
    uint32_t buf = 0, aph = 0;
    bool ok = true;
    for (long i = begin; i < end && ok;) {
      const int tile = (int)(i / wk.per_tile);
      const long tile_end = min(end, (long)(tile + 1) * wk.per_tile), share = blockIdx.x - wk.owner((long)tile * wk.per_tile, gridDim.x);
#pragma unroll
      for (int c = 0; c < L::kCols; ++c) sums[c] = 0.0f;
      for (; i < tile_end; ++i) {
        if (!tc::mbar_wait_warp(&acc_full[buf], aph)) { ok = false; break; }
        tc::tc_fence_after_sync();
        if (drains) {
          const uint32_t acc = tmem + buf * (uint32_t)L::kAcc + ((uint32_t)(q * 32) << 16) + half * L::kCols;
#pragma unroll
          for (int c = 0; c < L::kCols; c += 16) {
            uint32_t a[16], b[16];
            tc::tmem_ld_32(acc + c, a);
            tc::tmem_ld_32(acc + N + c, b);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[c + j] += __uint_as_float(a[j]) + __uint_as_float(b[j]);
          }
        }
        tc::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
        buf ^= 1u;
        aph ^= buf == 0;
      }
      if (ok && drains) {
        float* dst = wk.partial + ((long)tile * wk.slots_max + share) * (N * 128) + (half * L::kCols) * 128 + q * 32 + lane;
#pragma unroll
        for (int c = 0; c < L::kCols; ++c) dst[c * 128] = sums[c];
      }
    }
    if (!ok && lane == 0) atomicExch(err_flag, tc::kErrEpilogueWait);
  }
  tc::tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after_sync();
    tc::tmem_dealloc(tmem, L::kTmem);
  }
}

// h = act(a) u of the shares' sums.  A block: four rows of x, a tile's 64 columns.
__global__ void __launch_bounds__(256)
gated_shares_kernel(const Work wk, int rows /*of a share*/, long ctas, float* __restrict__ h, float* __restrict__ pre_gate, float* __restrict__ pre_up, int m, int n,
                    int act) {
  NRS_PDL_PROLOGUE();
  const int tile = blockIdx.x, r = blockIdx.y * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63;
  __shared__ int s_shares;   // (one thread's divisions)
  if (threadIdx.x == 0) {
    const long first = (long)tile * wk.per_tile;
    s_shares = (int)(wk.owner(first + wk.per_tile - 1, ctas) - wk.owner(first, ctas)) + 1;
  }
  __syncthreads();
  const int col = tile * 64 + c;
  if (r >= m || col >= n) return;
  const float* src = wk.partial + (long)tile * wk.slots_max * (rows * 128) + r * 128 + c;
  float a = 0.0f, u = 0.0f;
#pragma unroll 4
  for (int s = 0; s < s_shares; ++s) {
    a += src[(long)s * (rows * 128)];
    u += src[(long)s * (rows * 128) + 64];
  }
  const size_t at = (size_t)r * n + col;
  if (pre_gate) { pre_gate[at] = a; pre_up[at] = u; }
  h[at] = gated::act(a, act) * u;
}

template <int N>
int run(nrs_ctx* ctx, const Shape& s, const float* x, const float* wg, const float* wu, float* h, float* pg, float* pu) {
  using L = Layout<N>;
  CUtensorMap g, u, t;
  const uint64_t wdim[2] = {(uint64_t)s.n, (uint64_t)s.k}, wstr[1] = {(uint64_t)s.n}, xdim[2] = {(uint64_t)s.k, (uint64_t)s.m}, xstr[1] = {(uint64_t)s.k};
  const uint32_t wbox[2] = {32, kSlice}, xbox[2] = {kSlice, (uint32_t)N};
  const bool ok = tc::encode_tmap(&g, wg, false, 2, wdim, wstr, wbox, true) && tc::encode_tmap(&u, wu, false, 2, wdim, wstr, wbox, true) &&
                  tc::encode_tmap(&t, x, false, 2, xdim, xstr, xbox);
  NRS_REQUIRE(ctx, ok, NRS_ERR_CUDA, "gated layer: cuTensorMapEncodeTiled failed (%d x %d x %d)", s.m, s.n, s.k);
  Work wk{};
  wk.per_tile = (s.k + kSlice - 1) / kSlice;
  const long tiles = (s.n + 63) / 64;
  wk.total = tiles * wk.per_tile;
  // At least two slices a CTA.
  const long ctas = std::min<long>(ctx->sm_count, std::max<long>(1, wk.total / 2)), least = wk.total / ctas;
  wk.slots_max = (int)((wk.per_tile + least - 1) / least + 1);
  const size_t scratch = sizeof(float) * tiles * wk.slots_max * N * 128;
  if (scratch > ((size_t)256 << 20)) return NRS_ERR_UNSUPPORTED;   // (hundreds of thousands of columns)
  void* p = nullptr;
  int st = nrs_ws_slot(ctx, NRS_WS_PARTIAL, scratch, &p);
  if (st != NRS_OK) return st;
  wk.partial = (float*)p;
  int* err = nullptr;
  st = nrs_err_flag(ctx, &err);
  if (st != NRS_OK) return st;
  static NrsSmemAttr attr;
  NRS_ENSURE_SMEM(ctx, attr, gated_skinny_kernel<N>, L::kBytes);
  NrsProfScope prof(ctx, NRS_PROF_GEMM, 4.0 * s.m * s.n * s.k);
  NRS_PDL_LAUNCH(gated_skinny_kernel<N>, (unsigned)ctas, kThreads, L::kBytes, ctx->stream, g, u, t, wk, err);
  NRS_LAUNCHED(ctx);
  NRS_PDL_LAUNCH(gated_shares_kernel, dim3((unsigned)tiles, (unsigned)((s.m + 3) / 4)), 256, 0, ctx->stream, wk, N, ctas, h, pg, pu, s.m, s.n, s.act);
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

}  // namespace

int nrs_gated_skinny_fwd(nrs_ctx* ctx, const Shape& s, const float* x, const float* wg, const float* wu, float* h, float* pre_gate, float* pre_up) {
  const bool whole = s.n % 4 == 0 && s.k % 4 == 0 && (((uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu) & 15) == 0;   // TMA's strides and addresses
  if (ctx->math_mode != NRS_MATH_3XTF32 || !whole || !tc::tensor_map_encoder() || s.m > 128 || s.n > (1 << 28)) return NRS_ERR_UNSUPPORTED;
  if (s.m <= 16) return run<16>(ctx, s, x, wg, wu, h, pre_gate, pre_up);
  if (s.m <= 32) return run<32>(ctx, s, x, wg, wu, h, pre_gate, pre_up);
  if (s.m <= 64) return run<64>(ctx, s, x, wg, wu, h, pre_gate, pre_up);
  return run<128>(ctx, s, x, wg, wu, h, pre_gate, pre_up);
}
