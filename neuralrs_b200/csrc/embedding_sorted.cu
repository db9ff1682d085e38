// Embedding lookup with a scale, and the table's gradient from tokens sorted by their ids.
//
//   out[t, :] = scale * weight[id_t, :] (+ pos[t % seq, :])
//   dweight[v, :] (+)= scale * sum over the tokens with id_t = v, in the order of t, of g[t, :]
//
// Lookup as in the reference's embed_forward (src/cuda/nn/embedding.rs:13-21), which has no scale.  Its gradient adds every
// token's row with atomics (:23-30); the form in transformer.cu gives every vocabulary row a block that looks through all
// tokens, vocab * tokens comparisons.  Here two launches do tokens' work alone:
//
//   sort   every block owns a range of the vocabulary and looks through all ids (they stay in L2), a stretch of them a warp.
//          It counts those below its range, which is where its own start in the sorted order, and for each of its rows
//          and each warp the tokens there; the counts' running sums are the places, and a second look puts the tokens
//          there, (id, token) by (id, token).  No block needs another, and no warp waits for one, also not where one id
//          makes up most of the tokens.
//   sum    the sorted tokens are cut into equal pieces, so a token that makes up a tenth of the text costs no block more
//          than its share.  A run inside one piece goes straight to its row; one that crosses pieces leaves partial sums,
//          and the last of its blocks to finish adds them up, in order.  Other blocks among these write zeros to the rows
//          that no token has: the sums wait for memory much, zeros not at all.  (Zeros by the sorting blocks beside their
//          sort starve its loads: 16384 tokens x 1024 over 50000 rows 43 us for that launch, 36 for zeros behind it.)
//
// Deterministic: every sum has one order, whatever the blocks' timing.  Bound by memory: g read once, dweight written once.
#include <algorithm>

#include "igemm_problems.cuh"
#include "nrs_internal.h"

namespace {

constexpr int kErrBadIndex = 5;

// ------------------------------------------------------------------------------------------------ lookup

// One vector (VEC: 16 bytes) of a row per thread and step, four under way together.  WIDE: more of them than fast division
// takes.
template <bool VEC, bool WIDE>
__global__ void __launch_bounds__(256)
embed_scaled_kernel(const float* __restrict__ w, const int32_t* __restrict__ idx, const float* __restrict__ pos, float* __restrict__ out, size_t total,
                    int width /*vectors of a row*/, NrsFastDiv by_width, NrsFastDiv by_seq, int vocab, float scale, int* err) {
  NRS_PDL_PROLOGUE();
  constexpr int kDeep = 4;
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  for (size_t i0 = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i0 < total; i0 += kDeep * stride) {
    float4 v[kDeep], p[kDeep];
    uint32_t t[kDeep], c[kDeep];
    int row[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const size_t i = min(i0 + k * stride, total - 1);   // (past the end: the last one again)
      if (WIDE) {
        t[k] = (uint32_t)(i / (size_t)width);
        c[k] = (uint32_t)(i - (size_t)t[k] * width);
      } else {
        by_width.divmod((uint32_t)i, t[k], c[k]);
      }
      row[k] = idx[t[k]];
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      v[k] = p[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (row[k] >= 0 && row[k] < vocab) {
        const size_t at = (size_t)row[k] * width + c[k];
        if (VEC) v[k] = reinterpret_cast<const float4*>(w)[at];
        else v[k].x = w[at];
      } else if (c[k] == 0) {
        atomicExch(err, kErrBadIndex);
      }
      if (pos) {
        uint32_t q, r;
        by_seq.divmod(t[k], q, r);
        const size_t at = (size_t)r * width + c[k];
        if (VEC) p[k] = reinterpret_cast<const float4*>(pos)[at];
        else p[k].x = pos[at];
      }
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const size_t i = i0 + k * stride;
      if (i >= total) break;
      if (VEC) reinterpret_cast<float4*>(out)[i] = make_float4(fmaf(scale, v[k].x, p[k].x), fmaf(scale, v[k].y, p[k].y), fmaf(scale, v[k].z, p[k].z),
                                                               fmaf(scale, v[k].w, p[k].w));
      else out[i] = fmaf(scale, v[k].x, p[k].x);
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMaxRange = 1024;           // most vocabulary rows of a block: a count for each of them and each warp is 128 KB
constexpr int kSumWarps = 8;              // of a block that sums
constexpr int kSlab = 128;                // its columns
constexpr int kZeroRows = 64;             // vocabulary rows of a block that writes zeros
constexpr int kFillBlocks = 592;          // four for each of 148 SMs: fewer and pieces are made smaller

struct Plan {
  int tokens, dim, vocab, range;      // range: vocabulary rows of a sorting block
  int slabs, per_warp, pieces;        // sum: slabs of a row, tokens of a warp, pieces of the sorted tokens
  __host__ __device__ int piece() const { return kSumWarps * per_warp; }
};
Plan plan_of(int tokens, int dim, int vocab, int sm_count) {
  Plan p{tokens, dim, vocab, 0, (dim - 1) / kSlab + 1, 32, 0};
  p.range = std::min(kMaxRange, (vocab + sm_count - 1) / sm_count);
  while (p.per_warp > 4 && (long)((tokens + p.piece() - 1) / p.piece()) * p.slabs < kFillBlocks) p.per_warp /= 2;
  p.pieces = (tokens + p.piece() - 1) / p.piece();
  return p;
}
struct Work {            // in the caller's workspace, in this order
  int2* sorted;          // [tokens] (id, token)
  float* partial;        // [pieces][2][dim] sums of a piece's tokens whose run came from before it, and of those whose run goes on
  unsigned* tickets;     // [pieces][slabs] how many pieces of the run that starts in a piece are done
  int* start;            // [vocab + 1] first sorted token of each row
};
size_t work_of(const Plan& p, void* base, Work* w) {
  uint8_t* at = (uint8_t*)base;
  size_t used = 0;
  auto take = [&](size_t bytes) {
    void* q = at + used;
    used += (bytes + 255) / 256 * 256;
    return q;
  };
  Work x;
  x.sorted = (int2*)take(sizeof(int2) * p.tokens);
  x.partial = (float*)take(sizeof(float) * 2 * p.pieces * p.dim);
  x.tickets = (unsigned*)take(sizeof(unsigned) * p.pieces * p.slabs);
  x.start = (int*)take(sizeof(int) * ((size_t)p.vocab + 1));
  if (w) *w = x;
  return used;
}

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_scan(int v, int lane) {   // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}
__global__ void __launch_bounds__(kSortThreads, 1)
embed_sort_kernel(const int32_t* __restrict__ idx, const Plan p, const Work w) {
  NRS_PDL_PROLOGUE();
  // (All of it dynamic: whether a launch has to ask for more than the default is judged by that size alone.)
  extern __shared__ int s_below[];                 // [warp]
  int* const s_scan = s_below + kSortWarps;        // [warp]
  int* const counts = s_scan + kSortWarps;         // [warp][range] tokens of each row in the warp's stretch, then where its next goes
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lo = blockIdx.x * p.range, hi = min(p.vocab, lo + p.range), rows = hi - lo;
  int* const mine = counts + warp * p.range;
  // A warp's tokens: a stretch of its own, so the warps go through them without waiting for each other.
  const int stretch = (p.tokens + kSortWarps - 1) / kSortWarps;
  const int begin = (int)min((long)p.tokens, (long)warp * stretch), stop = (int)min((long)p.tokens, (long)begin + stretch);
  for (int r = lane; r < rows; r += 32) mine[r] = 0;
  for (long i = (long)blockIdx.x * kSortThreads + tid; i < (long)p.pieces * p.slabs; i += (long)gridDim.x * kSortThreads) w.tickets[i] = 0;
  __syncwarp();

  // How many tokens each row has, and how many lie below the range.  (Ids outside the vocabulary are nobody's.)
  constexpr int kDeep = 8;                         // loads under way together
  int below = 0;
  for (int t0 = begin + lane; t0 < stop; t0 += 32 * kDeep) {
    int id[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) id[k] = t0 + 32 * k < stop ? idx[t0 + 32 * k] : -1;
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      below += id[k] >= 0 && id[k] < lo;
      if (id[k] >= lo && id[k] < hi) atomicAdd(&mine[id[k] - lo], 1);
    }
  }
  below = warp_sum(below);
  if (lane == 0) s_below[warp] = below;
  __syncthreads();
  const int first = warp_sum(s_below[lane]);       // where the range starts in the sorted order

  // Counts to places: a row a thread, its warps' tokens behind each other, the rows likewise.
  int total = 0;
  if (tid < rows) {
#pragma unroll 8
    for (int k = 0; k < kSortWarps; ++k) {
      const int c = counts[k * p.range + tid];
      counts[k * p.range + tid] = total;
      total += c;
    }
  }
  const int incl = warp_scan(total, lane);
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  const int start = first + warp_sum(lane < warp ? s_scan[lane] : 0) + incl - total;
  if (tid < rows) {
    w.start[lo + tid] = start;
#pragma unroll 8
    for (int k = 0; k < kSortWarps; ++k) counts[k * p.range + tid] += start;
  }
  if (hi == p.vocab && tid == rows - 1) w.start[p.vocab] = start + total;
  __syncthreads();

  // Each token behind those of its id that came before it, 32 at a time.
  for (int t0 = begin; t0 < stop; t0 += 32 * kDeep) {
    int id[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) id[k] = t0 + 32 * k + lane < stop ? idx[t0 + 32 * k + lane] : -1;
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const bool hit = id[k] >= lo && id[k] < hi;
      if (!__any_sync(0xffffffffu, hit)) continue;
      const unsigned same = __match_any_sync(0xffffffffu, hit ? id[k] : -1);
      const int rank = __popc(same & ((1u << lane) - 1u)), to = hit ? mine[id[k] - lo] + rank : 0;
      __syncwarp();
      if (hit) {
        w.sorted[to] = make_int2(id[k], t0 + 32 * k + lane);
        if (rank == 0) mine[id[k] - lo] = to + __popc(same);
      }
      __syncwarp();
    }
  }
}

// ------------------------------------------------------------------------------------------------ sum

// A lane's four columns of a slab: neighbours (VEC), or 32 apart.
template <bool VEC>
struct Cols {
  int c0, dim;
  __device__ __forceinline__ void load(float (&v)[4], const float* row) const {
    if (VEC) {
      const float4 q = c0 < dim ? *reinterpret_cast<const float4*>(row + c0) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c0 + 32 * j < dim ? row[c0 + 32 * j] : 0.0f;
    }
  }
  // The same of what another block has written.
  __device__ __forceinline__ void load_shared(float (&v)[4], const float* row) const {
    if (VEC) {
      const float4 q = c0 < dim ? __ldcg(reinterpret_cast<const float4*>(row + c0)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c0 + 32 * j < dim ? __ldcg(row + c0 + 32 * j) : 0.0f;
    }
  }
  __device__ __forceinline__ void store(const float (&v)[4], float* row) const {
    if (VEC) {
      if (c0 < dim) *reinterpret_cast<float4*>(row + c0) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + 32 * j < dim) row[c0 + 32 * j] = v[j];
    }
  }
};

template <bool VEC>
__global__ void __launch_bounds__(kSumWarps * 32)
embed_sum_kernel(const float* __restrict__ g, const Plan p, const Work w, float* dw, float scale, int accumulate, unsigned zero_blocks) {
  NRS_PDL_PROLOGUE();
  // The blocks that write zeros are spread among those that sum.
  const unsigned zeros_before = (unsigned)((uint64_t)blockIdx.x * zero_blocks / gridDim.x);
  if ((unsigned)((uint64_t)(blockIdx.x + 1) * zero_blocks / gridDim.x) != zeros_before) {
    const int r0 = (int)zeros_before * kZeroRows, r1 = min(p.vocab, r0 + kZeroRows);
    for (int r = r0 + (threadIdx.x >> 5); r < r1; r += kSumWarps) {
      if (w.start[r] != w.start[r + 1]) continue;
      float* row = dw + (size_t)r * p.dim;
      if (VEC)
        for (int c = threadIdx.x & 31; c < p.dim / 4; c += 32) reinterpret_cast<float4*>(row)[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      else
        for (int c = threadIdx.x & 31; c < p.dim; c += 32) row[c] = 0.0f;
    }
    return;
  }
  const unsigned block = blockIdx.x - zeros_before;
  __shared__ float4 s_head[kSumWarps][32], s_tail[kSumWarps][32];
  __shared__ int s_last[2];                        // ids whose pieces' sums this block adds up
  __shared__ int s_flags[kSumWarps];               // 1: has a sum for a run from before; 2: for one that goes on; 4: both are one run
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int piece = block / p.slabs, slab = block - piece * p.slabs;
  const Cols<VEC> cols{slab * kSlab + (VEC ? 4 * lane : lane), p.dim};
  const int base = piece * p.piece() + warp * p.per_warp;
  // (loaded together: the pairs behind the last valid one are not looked at)
  const int edge_at = lane == 0 ? base - 1 : base + p.per_warp;
  const int2 pair = base + lane < p.tokens && lane < p.per_warp ? w.sorted[base + lane] : make_int2(-1, 0);
  const int beside = lane < 2 && edge_at >= 0 && edge_at < p.tokens ? w.sorted[edge_at].x : -1;
  const int valid = w.start[p.vocab], n = min(p.per_warp, valid - base);   // valid: tokens with an id of the vocabulary

  auto finish = [&](int id, const float (&a)[4]) {   // a row's sum is complete
    float* row = dw + (size_t)id * p.dim;
    float r[4];
    if (accumulate) {
      cols.load(r, row);
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = fmaf(scale, a[j], r[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = scale * a[j];
    }
    cols.store(r, row);
  };

  int flags = 0, id_first = -1, id_last = -1;
  if (n > 0) {
    const int2 e = lane < n ? pair : make_int2(-1, 0);
    const int edge = lane == 1 && base + n >= valid ? -1 : beside;
    id_first = __shfl_sync(0xffffffffu, e.x, 0);
    id_last = __shfl_sync(0xffffffffu, e.x, n - 1);
    const bool from_before = __shfl_sync(0xffffffffu, edge, 0) == id_first, goes_on = __shfl_sync(0xffffffffu, edge, 1) == id_last;
    float acc[4] = {};
    int id = id_first;
    bool first_run = true;
    constexpr int kDeep = 8;
    for (int i0 = 0; i0 < n; i0 += kDeep) {
      float v[kDeep][4];
#pragma unroll
      for (int k = 0; k < kDeep; ++k) {
        if (i0 + k >= n) break;
        cols.load(v[k], g + (size_t)__shfl_sync(0xffffffffu, e.y, i0 + k) * p.dim);
      }
#pragma unroll
      for (int k = 0; k < kDeep; ++k) {
        if (i0 + k >= n) break;
        const int now = __shfl_sync(0xffffffffu, e.x, i0 + k);
        if (now != id) {
          if (first_run && from_before) {
            s_head[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            flags |= 1;
          } else {
            finish(id, acc);
          }
          first_run = false;
          id = now;
          acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += v[k][j];
      }
    }
    const bool head = first_run && from_before;
    if (head) {
      s_head[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      flags |= goes_on ? 5 : 1;
    } else if (goes_on) {
      s_tail[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      flags |= 2;
    } else {
      finish(id, acc);
    }
  }
  if (lane == 0) s_flags[warp] = flags;
  if (threadIdx.x < 2) s_last[threadIdx.x] = -1;
  __syncthreads();

  // The sums of one run that lie in several warps: added up by the warp where it starts, or (a run from an earlier piece)
  // the first.  A warp may have two such runs.
  auto chain = [&](bool incoming) {
    const int id = incoming ? id_first : id_last;
    const float4 q = incoming ? s_head[warp][lane] : s_tail[warp][lane];
    float a[4] = {q.x, q.y, q.z, q.w};
    bool on = incoming ? (flags & 4) != 0 : true;  // the run goes on behind this warp
    for (int k = warp + 1; on && k < kSumWarps; ++k) {
      const float4 o = s_head[k][lane];
      a[0] += o.x; a[1] += o.y; a[2] += o.z; a[3] += o.w;
      on = (s_flags[k] & 4) != 0;
    }
    if (!incoming && !on) {
      finish(id, a);
      return;
    }
    // The run crosses pieces: the last of them to get here adds their sums up, in order.
    const int from = w.start[id] / p.piece(), to = (w.start[id + 1] - 1) / p.piece();
    cols.store(a, w.partial + ((size_t)piece * 2 + (incoming ? 0 : 1)) * p.dim);
    __threadfence();
    __syncwarp();
    if (lane == 0 && atomicAdd(&w.tickets[(size_t)from * p.slabs + slab], 1u) == (unsigned)(to - from)) {
      s_last[incoming ? 0 : 1] = id;
      __threadfence();
    }
  };
  if (warp == 0 && (flags & 1)) chain(true);
  if (flags & 2) chain(false);
  __syncthreads();
  // Such a sum: every warp adds a stretch of the pieces, the first the stretches.  (By one warp the 512 pieces of a token that
  // is everywhere take 44 us.)
  for (int which = 0; which < 2; ++which) {
    const int id = s_last[which];
    if (id < 0) continue;
    const int from = w.start[id] / p.piece(), to = (w.start[id + 1] - 1) / p.piece(), each = (to - from + kSumWarps) / kSumWarps;
    const int k0 = from + warp * each, k1 = min(to + 1, k0 + each);
    float a[4] = {};
    constexpr int kDeep = 8;
    for (int k = k0; k < k1; k += kDeep) {
      float v[kDeep][4];
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        if (k + i >= k1) break;
        cols.load_shared(v[i], w.partial + ((size_t)(k + i) * 2 + (k + i == from ? 1 : 0)) * p.dim);
      }
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        if (k + i >= k1) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] += v[i][j];
      }
    }
    s_head[warp][lane] = make_float4(a[0], a[1], a[2], a[3]);
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int k = 1; k < kSumWarps; ++k) {
        const float4 o = s_head[k][lane];
        a[0] += o.x; a[1] += o.y; a[2] += o.z; a[3] += o.w;
      }
      finish(id, a);
    }
    __syncthreads();
  }
}

}  // namespace

extern "C" {

int nrs_embedding_scaled_fwd(nrs_ctx* ctx, const float* weight, const int32_t* idx, const float* pos_table, float* out, int tokens, int seq, int dim,
                             int vocab, float scale) {
  NRS_REQUIRE_CTX(ctx);
  NRS_REQUIRE(ctx, tokens >= 0 && dim > 0 && vocab > 0, NRS_ERR_SHAPE, "%s: bad shape [%d,%d], vocabulary %d", __func__, tokens, dim, vocab);
  NRS_REQUIRE(ctx, !pos_table || seq > 0, NRS_ERR_SHAPE, "%s: sequence length must be positive", __func__);
  if (tokens == 0) return NRS_OK;
  NRS_REQUIRE(ctx, weight && idx && out, NRS_ERR_ARG, "%s: null tensor", __func__);
  NrsDeviceGuard on(ctx);
  int* err = nullptr;
  const int st = nrs_err_flag(ctx, &err);
  if (st != NRS_OK) return st;
  const bool vec = dim % 4 == 0 && (((uintptr_t)weight | (uintptr_t)out | (uintptr_t)pos_table) & 15) == 0;
  const int width = vec ? dim / 4 : dim;
  const size_t total = (size_t)tokens * width, want = (total + 255) / 256, cap = (size_t)ctx->sm_count * 16;
  const unsigned blocks = (unsigned)(want < cap ? want : cap);
  const bool wide = total > 0x7fffffffu;
  const NrsFastDiv by_width(width), by_seq(pos_table ? seq : 1);
#define NRS_EMBED(VEC_, WIDE_) \
  NRS_PDL_LAUNCH((embed_scaled_kernel<VEC_, WIDE_>), blocks, 256, 0, ctx->stream, weight, idx, pos_table, out, total, width, by_width, by_seq, vocab, scale, err)
  if (vec && !wide) NRS_EMBED(true, false);
  else if (vec) NRS_EMBED(true, true);
  else if (!wide) NRS_EMBED(false, false);
  else NRS_EMBED(false, true);
#undef NRS_EMBED
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

size_t nrs_embedding_sorted_workspace(int tokens, int dim, int vocab) {
  if (tokens < 0 || dim <= 0 || vocab <= 0) return 0;
  return work_of(plan_of(tokens, dim, vocab, 1), nullptr, nullptr);
}

int nrs_embedding_sorted_bwd(nrs_ctx* ctx, const float* g, const int32_t* idx, float* dweight, int tokens, int dim, int vocab, float scale, int accumulate,
                             void* workspace, size_t workspace_bytes) {
  NRS_REQUIRE_CTX(ctx);
  NRS_REQUIRE(ctx, tokens >= 0 && dim > 0 && vocab > 0 && tokens <= (1 << 30) && vocab <= (1 << 30), NRS_ERR_SHAPE, "%s: bad shape [%d,%d], vocabulary %d", __func__, tokens, dim, vocab);
  if (tokens == 0 && accumulate) return NRS_OK;
  NRS_REQUIRE(ctx, dweight && (tokens == 0 || (g && idx)), NRS_ERR_ARG, "%s: null tensor", __func__);
  const Plan p = plan_of(tokens, dim, vocab, ctx->sm_count);
  Work w{};
  const size_t need = work_of(p, workspace, &w);
  NRS_REQUIRE(ctx, workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, NRS_ERR_ARG,
              "%s: needs a workspace of %zu bytes on a 16-byte boundary", __func__, need);
  NRS_REQUIRE(ctx, (long)p.pieces * p.slabs + vocab <= 0x7fffffffL, NRS_ERR_SHAPE, "%s: %d tokens of %d features are too many for one call", __func__, tokens, dim);
  NrsDeviceGuard on(ctx);
  const bool vec = dim % 4 == 0 && (((uintptr_t)g | (uintptr_t)dweight) & 15) == 0;
  const size_t smem = sizeof(int) * kSortWarps * (p.range + 2);
  static NrsSmemAttr attr;
  NRS_ENSURE_SMEM(ctx, attr, embed_sort_kernel, smem);
  NRS_PDL_LAUNCH(embed_sort_kernel, (vocab + p.range - 1) / p.range, kSortThreads, smem, ctx->stream, idx, p, w);
  NRS_LAUNCHED(ctx);
  const unsigned zeros = accumulate ? 0 : (unsigned)((vocab + kZeroRows - 1) / kZeroRows), blocks = (unsigned)(p.pieces * p.slabs) + zeros;
  if (vec) NRS_PDL_LAUNCH(embed_sum_kernel<true>, blocks, kSumWarps * 32, 0, ctx->stream, g, p, w, dweight, scale, accumulate != 0, zeros);
  else NRS_PDL_LAUNCH(embed_sum_kernel<false>, blocks, kSumWarps * 32, 0, ctx->stream, g, p, w, dweight, scale, accumulate != 0, zeros);
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

}  // extern "C"
