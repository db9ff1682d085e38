// Norms of query and key heads with the rotation of their positions in the same pass, forward and backward.  No reference
// counterpart (its attention adds a sinusoidal table to the embedding, src/cuda/nn/positional.rs:18-44).
//
// Per token and head, x of d features, rstd = 1 / sqrt(mean(x^2) + eps):
//   z = gamma x rstd,   y = R z,   R turning each pair (a, b) of the first `rot` features by the angle of the token's
//   position: (a cos - b sin, a sin + b cos)
//   backward: dz = R^T g,   dx = rstd (gamma dz - x rstd^2 mean(gamma dz x)),   dgamma = sum over tokens and heads of dz x rstd
// All sums in f32: d terms in one fixed order by shuffles; dgamma per thread over its rows, then over a block's threads, then
// over the blocks, in fixed order without atomics.
//
// Bound by memory: 8 bytes a feature forward, 12 backward.  A row is held in the registers of L neighbouring lanes, eight
// features each in two 16-byte accesses, placed so that a lane holds both members of its pairs: nothing but the row sum
// crosses lanes.  A warp's rows are heads side by side, of one token or of several; each looks up its own position and angles,
// which the caches keep for the token's other heads.
#include <algorithm>

#include "igemm_problems.cuh"
#include "nrs_internal.h"

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kDeep = 2;                            // rows of a lane under way together
constexpr int kBlocksFwd = 3, kBlocksBwd = 2;       // blocks an SM, all of them resident
constexpr int kErrBadPosition = 6;
constexpr int kMaxHead = 1024;

struct Side {   // of the queries, or of the keys
  const float* x;
  const float* g;       // backward
  const float* gamma;   // null: ones
  float* y;             // forward: the result; backward: dx, or null
  float* partial;       // backward: [blocks of this side][d], or null
  long ld_x, ld_g, ld_y;
  int heads;
  int first_block, blocks;
  NrsFastDiv div;       // of heads
};
struct Args {
  Side side[2];
  const float* table;     // [max_len][rot / 2][cos, sin], or null
  const int32_t* pos;     // or null: t % seq
  int* err;
  int tokens, seq, d, rot, max_len, accumulate;
  NrsFastDiv div_seq;
  float eps, inv_d;
};

__device__ __forceinline__ int token_of(long i, int per) { return i >> 32 ? (int)(i / per) : (int)((uint32_t)i / (uint32_t)per); }

// The position of token t, or -1 outside the table.
__device__ __forceinline__ int position(const Args& a, int t) {
  if (!a.table) return 0;
  int p;
  if (a.pos) {
    p = a.pos[t];
  } else {
    uint32_t q, r;
    a.div_seq.divmod((uint32_t)t, q, r);
    p = (int)r;
  }
  return p >= 0 && p < a.max_len ? p : -1;
}

// (x, y) turned by the angle of (c, s)
__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
  const float a = x * c - y * s, b = x * s + y * c;
  x = a;
  y = b;
}

// Eight features of a lane: A at offset oa, B at ob.  Not interleaved: (A.i, B.i) are pairs; interleaved: the neighbours
// inside A and inside B.  `back`: R^T.
template <bool INTER>
__device__ __forceinline__ void rotate(float (&A)[4], float (&B)[4], const float4& t0, const float4& t1, bool back) {
  const float sg = back ? -1.0f : 1.0f;
  if (INTER) {
    turn(A[0], A[1], t0.x, sg * t0.y);
    turn(A[2], A[3], t0.z, sg * t0.w);
    turn(B[0], B[1], t1.x, sg * t1.y);
    turn(B[2], B[3], t1.z, sg * t1.w);
  } else {
    turn(A[0], B[0], t0.x, sg * t0.y);
    turn(A[1], B[1], t0.z, sg * t0.w);
    turn(A[2], B[2], t1.x, sg * t1.y);
    turn(A[3], B[3], t1.z, sg * t1.w);
  }
}

template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int d = L / 2; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ __forceinline__ void get(float (&v)[4], const float* p, bool on) {
  const float4 q = on ? *reinterpret_cast<const float4*>(p) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
__device__ __forceinline__ void put(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }

// L: lanes of a row.  d and rot are multiples of 8, d <= 8 * L, every row starts on 16 bytes.  A row is a token's head; a warp
// takes 32 / L of them side by side and kDeep times that together, so that their loads, and behind the positions those of the
// table, are all under way before the first sum.
template <int L, bool INTER, bool BWD>
__global__ void __launch_bounds__(kThreads, BWD ? kBlocksBwd : kBlocksFwd) head_norm_kernel(const Args a) {
  NRS_PDL_PROLOGUE();
  constexpr int R = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, u = lane % L, sub = lane / L;
  const bool keys = (int)blockIdx.x >= a.side[1].first_block;
  const Side& s = a.side[keys ? 1 : 0];
  const bool have = 8 * u < a.d, turns = 8 * u < a.rot;
  const int oa = turns ? 4 * u : 8 * u, ob = turns ? a.rot / 2 + 4 * u : 8 * u + 4;
  const int ta = INTER ? oa : 8 * u, tb = INTER ? ob : 8 * u + 4;   // of the table's row
  float wa[4], wb[4], da[4] = {}, db[4] = {};
  if (s.gamma) {
    get(wa, s.gamma + oa, have);
    get(wb, s.gamma + ob, have);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) wa[j] = wb[j] = 1.0f;
  }
  const uint32_t rows = (uint32_t)a.tokens * (uint32_t)s.heads, step = (uint32_t)s.blocks * (kWarps * R * kDeep);   // (the launcher checks the range)
  for (uint32_t r0 = ((uint32_t)((int)blockIdx.x - s.first_block) * kWarps + warp) * (R * kDeep); r0 < rows; r0 += step) {
    float A[kDeep][4], B[kDeep][4], GA[BWD ? kDeep : 1][4], GB[BWD ? kDeep : 1][4];
    float4 t0[kDeep], t1[kDeep];
    uint32_t t[kDeep], h[kDeep];
    int p[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const uint32_t r = r0 + k * R + sub;
      s.div.divmod(min(r, rows - 1), t[k], h[k]);
      const bool on = have && r < rows;
      const float* x = s.x + (size_t)t[k] * s.ld_x + h[k] * a.d;
      get(A[k], x + oa, on);
      get(B[k], x + ob, on);
      if (BWD) {
        const float* g = s.g + (size_t)t[k] * s.ld_g + h[k] * a.d;
        get(GA[BWD ? k : 0], g + oa, on);
        get(GB[BWD ? k : 0], g + ob, on);
      }
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      p[k] = position(a, t[k]);
      t0[k] = t1[k] = make_float4(1.0f, 0.0f, 1.0f, 0.0f);
      if (turns && p[k] >= 0) {
        const float* row = a.table + (size_t)p[k] * a.rot;
        t0[k] = *reinterpret_cast<const float4*>(row + ta);
        t1[k] = *reinterpret_cast<const float4*>(row + tb);
      }
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const uint32_t r = r0 + k * R + sub;
      const bool on = have && r < rows;
      if (p[k] < 0 && u == 0 && r < rows) atomicExch(a.err, kErrBadPosition);
      float sq = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) sq += A[k][j] * A[k][j] + B[k][j] * B[k][j];
      const float root = rsqrtf(row_sum<L>(sq) * a.inv_d + a.eps), rstd = r < rows && (!BWD || p[k] >= 0) ? root : 0.0f;   // (past the end, without an eps: no 0 * inf into dgamma)
      if (!BWD) {
        float* y = s.y + (size_t)t[k] * s.ld_y + h[k] * a.d;
#pragma unroll
        for (int j = 0; j < 4; ++j) { A[k][j] *= rstd * wa[j]; B[k][j] *= rstd * wb[j]; }
        if (turns) rotate<INTER>(A[k], B[k], t0[k], t1[k], false);
        if (p[k] < 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) A[k][j] = B[k][j] = 0.0f;
        }
        if (on) { put(y + oa, A[k]); put(y + ob, B[k]); }
      } else {
        float(&ga)[4] = GA[BWD ? k : 0];
        float(&gb)[4] = GB[BWD ? k : 0];
        if (p[k] < 0) {   // (whatever the row holds: the normed values below are 0, too)
#pragma unroll
          for (int j = 0; j < 4; ++j) A[k][j] = B[k][j] = ga[j] = gb[j] = 0.0f;
        }
        if (turns) rotate<INTER>(ga, gb, t0[k], t1[k], true);
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          A[k][j] *= rstd; B[k][j] *= rstd;                       // the normed values
          da[j] += ga[j] * A[k][j]; db[j] += gb[j] * B[k][j];
          ga[j] *= wa[j]; gb[j] *= wb[j];
          dot += ga[j] * A[k][j] + gb[j] * B[k][j];
        }
        const float mean = row_sum<L>(dot) * a.inv_d;
        if (on && s.y) {
          float* y = s.y + (size_t)t[k] * s.ld_y + h[k] * a.d;
          float ra[4], rb[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) { ra[j] = rstd * (ga[j] - A[k][j] * mean); rb[j] = rstd * (gb[j] - B[k][j] * mean); }
          if (a.accumulate) {
            float o[4];
            get(o, y + oa, true);
#pragma unroll
            for (int j = 0; j < 4; ++j) ra[j] += o[j];
            get(o, y + ob, true);
#pragma unroll
            for (int j = 0; j < 4; ++j) rb[j] += o[j];
          }
          put(y + oa, ra);
          put(y + ob, rb);
        }
      }
    }
  }
  if (BWD && s.partial) {
    __shared__ float sums[kWarps][8 * L];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int d = L; d < 32; d <<= 1) {
        da[j] += __shfl_xor_sync(0xffffffffu, da[j], d);
        db[j] += __shfl_xor_sync(0xffffffffu, db[j], d);
      }
    }
    if (sub == 0 && have) { put(&sums[warp][oa], da); put(&sums[warp][ob], db); }
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += kThreads) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += sums[w][c];
      s.partial[(size_t)((int)blockIdx.x - s.first_block) * a.d + c] = v;
    }
  }
}

// The same for any size and alignment: a warp per row, feature by feature, the row read twice (the second time from L1).
template <bool BWD>
__global__ void __launch_bounds__(kThreads) head_norm_any_kernel(const Args a, int interleaved) {
  NRS_PDL_PROLOGUE();
  extern __shared__ float acc[];      // backward: [warps][d]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool keys = (int)blockIdx.x >= a.side[1].first_block;
  const Side& s = a.side[keys ? 1 : 0];
  float* mine = acc + warp * a.d;
  if (BWD) {
    for (int c = lane; c < a.d; c += 32) mine[c] = 0.0f;
    __syncwarp();
  }
  const int half = a.rot / 2, units = a.d - half;   // a unit: a pair, or one feature behind them
  auto first = [&](int i) { return i < half ? (interleaved ? 2 * i : i) : i + half; };
  auto second = [&](int i) { return interleaved ? 2 * i + 1 : i + half; };
  auto w = [&](int c) { return s.gamma ? s.gamma[c] : 1.0f; };
  const long rows = (long)a.tokens * s.heads, step = (long)s.blocks * kWarps;
  for (long r = (long)((int)blockIdx.x - s.first_block) * kWarps + warp; r < rows; r += step) {
    const int t = token_of(r, s.heads), h = (int)(r - (long)t * s.heads);
    const int p = position(a, t);
    if (p < 0 && lane == 0) atomicExch(a.err, kErrBadPosition);
    const float* x = s.x + (size_t)t * s.ld_x + (size_t)h * a.d;
    const float* g = BWD ? s.g + (size_t)t * s.ld_g + (size_t)h * a.d : nullptr;
    float* y = s.y ? s.y + (size_t)t * s.ld_y + (size_t)h * a.d : nullptr;
    const float* row = a.table ? a.table + (size_t)max(p, 0) * a.rot : nullptr;
    // the gradient of the unit's z, before gamma
    auto unit = [&](const float* v, int i, float& e, float& f, bool back) {
      e = v[first(i)];
      f = i < half ? v[second(i)] : 0.0f;
      if (back && i < half) turn(e, f, row[2 * i], -row[2 * i + 1]);
    };
    if (BWD && p < 0) {                 // nothing of the row counts, whatever it holds
      for (int c = lane; y && !a.accumulate && c < a.d; c += 32) y[c] = 0.0f;
      continue;
    }
    float sq = 0.0f;
    for (int c = lane; c < a.d; c += 32) sq += x[c] * x[c];
    const float rstd = rsqrtf(row_sum<32>(sq) * a.inv_d + a.eps);
    if (!BWD) {
      for (int i = lane; i < units; i += 32) {
        float e, f;
        unit(x, i, e, f, false);
        e *= rstd * w(first(i));
        if (i < half) { f *= rstd * w(second(i)); turn(e, f, row[2 * i], row[2 * i + 1]); }
        y[first(i)] = p < 0 ? 0.0f : e;
        if (i < half) y[second(i)] = p < 0 ? 0.0f : f;
      }
      continue;
    }
    float dot = 0.0f;
    for (int i = lane; i < units; i += 32) {
      float ge, gf, xe, xf;
      unit(g, i, ge, gf, true);
      unit(x, i, xe, xf, false);
      xe *= rstd; xf *= rstd;
      mine[first(i)] += ge * xe;
      dot += ge * w(first(i)) * xe;
      if (i < half) { mine[second(i)] += gf * xf; dot += gf * w(second(i)) * xf; }
    }
    const float mean = row_sum<32>(dot) * a.inv_d;
    if (!y) continue;
    for (int i = lane; i < units; i += 32) {
      float ge, gf, xe, xf;
      unit(g, i, ge, gf, true);
      unit(x, i, xe, xf, false);
      const float e = rstd * (ge * w(first(i)) - xe * rstd * mean);
      const float f = i < half ? rstd * (gf * w(second(i)) - xf * rstd * mean) : 0.0f;
      float* pe = y + first(i);
      *pe = a.accumulate ? *pe + e : e;
      if (i < half) {
        float* pf = y + second(i);
        *pf = a.accumulate ? *pf + f : f;
      }
    }
  }
  if (BWD && s.partial) {
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += kThreads) {
      float v = 0.0f;
      for (int k = 0; k < kWarps; ++k) v += acc[k * a.d + c];
      s.partial[(size_t)((int)blockIdx.x - s.first_block) * a.d + c] = v;
    }
  }
}

// dgamma[c] (+)= the blocks' sums, for both sides.  32 columns a block; a warp adds every 32nd partial row.
__global__ void __launch_bounds__(1024)
head_norm_fold_kernel(const float* __restrict__ pq, int nq, float* dq, const float* __restrict__ pk, int nk, float* dk, int d, int accumulate) {
  NRS_PDL_PROLOGUE();
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const float* src = blockIdx.y ? pk : pq;
  float* dst = blockIdx.y ? dk : dq;
  if (!dst) return;
  const int n = blockIdx.y ? nk : nq;
  float v = 0.0f;
  if (c < d)
    for (int b = warp; b < n; b += 32) v += src[(size_t)b * d + c];
  sums[warp][lane] = v;
  __syncthreads();
  v = row_sum<32>(sums[lane][warp]);   // of column `warp`
  if (lane == 0 && blockIdx.x * 32 + warp < d) {
    float* o = dst + blockIdx.x * 32 + warp;
    *o = accumulate ? *o + v : v;
  }
}

// cos and sin of pos * base^(-2i / rot): the angle in 64 bits (in 32 a position of 1e5 would be off by 4e-3 of a turn)
__global__ void __launch_bounds__(256) rotary_table_kernel(float* __restrict__ table, int max_len, int half, double base) {
  NRS_PDL_PROLOGUE();
  const size_t n = (size_t)max_len * half, stride = (size_t)gridDim.x * blockDim.x;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += stride) {
    const size_t p = i / half;
    double s, c;
    sincos((double)p * pow(base, -(double)(i - p * half) / (double)half), &s, &c);
    table[2 * i] = (float)c;
    table[2 * i + 1] = (float)s;
  }
}

// Blocks of the two sides: enough for their rows, at most as many as are resident, shared out by the sides' rows.
void plan_blocks(const nrs_ctx* ctx, Args* a, int per_block, int per_sm) {
  const long cap = (long)ctx->sm_count * per_sm;
  long want[2];
  for (int i = 0; i < 2; ++i) want[i] = ((long)a->tokens * a->side[i].heads + per_block - 1) / per_block;
  if (want[0] + want[1] > cap) {
    long q = want[0] ? std::max(1L, cap * want[0] / (want[0] + want[1])) : 0;
    if (want[1]) q = std::min(q, cap - 1);
    want[1] = std::min(want[1], cap - q);
    want[0] = q;
  }
  for (int i = 0, at = 0; i < 2; at += a->side[i++].blocks) {
    a->side[i].first_block = at;
    a->side[i].blocks = (int)want[i];
  }
}

int lanes_of(int d) {
  int l = 1;
  while (8 * l < d) l <<= 1;
  return l < 4 ? 4 : l > 32 ? 32 : l;
}

struct Shape { int tokens, seq, heads_q, heads_k, d, rot, max_len, interleaved; float eps; };

int check_shape(nrs_ctx* ctx, const char* who, const Shape& s, const float* table, const int32_t* positions) {
  NRS_REQUIRE(ctx, s.tokens >= 0 && s.heads_q >= 0 && s.heads_k >= 0 && s.d > 0, NRS_ERR_SHAPE, "%s: bad shape: %d tokens, %d and %d heads of %d", who,
              s.tokens, s.heads_q, s.heads_k, s.d);
  NRS_REQUIRE(ctx, (long)s.heads_q * s.d <= 0x7fffffffL && (long)s.heads_k * s.d <= 0x7fffffffL, NRS_ERR_SHAPE, "%s: a row of %d or %d heads of %d", who, s.heads_q,
              s.heads_k, s.d);
  NRS_REQUIRE(ctx, s.d <= kMaxHead, NRS_ERR_UNSUPPORTED, "%s: heads of %d features (at most %d)", who, s.d, kMaxHead);
  NRS_REQUIRE(ctx, s.eps >= 0.0f, NRS_ERR_ARG, "%s: negative eps", who);
  if (!table) {
    NRS_REQUIRE(ctx, s.rot == 0, NRS_ERR_ARG, "%s: a rotation of %d features needs a table", who, s.rot);
    return NRS_OK;
  }
  NRS_REQUIRE(ctx, s.rot > 0 && s.rot % 2 == 0 && s.rot <= s.d, NRS_ERR_SHAPE, "%s: %d of %d features cannot rotate in pairs", who, s.rot, s.d);
  NRS_REQUIRE(ctx, s.max_len > 0, NRS_ERR_SHAPE, "%s: empty rotation table", who);
  if (!positions) {
    NRS_REQUIRE(ctx, s.seq > 0, NRS_ERR_SHAPE, "%s: sequence length must be positive", who);
    NRS_REQUIRE(ctx, (s.seq < s.tokens ? s.seq : s.tokens) <= s.max_len, NRS_ERR_SHAPE, "%s: sequence longer than the rotation table (%d > %d)", who,
                s.seq < s.tokens ? s.seq : s.tokens, s.max_len);
  }
  return NRS_OK;
}

// The tensors of one side.  (A side without heads takes no part.)
int check_side(nrs_ctx* ctx, const char* who, const char* which, const Side& s, int d, bool bwd) {
  if (s.heads == 0) return NRS_OK;
  NRS_REQUIRE(ctx, s.x && (bwd ? s.g != nullptr : s.y != nullptr), NRS_ERR_ARG, "%s: null tensor (%s)", who, which);
  const long row = (long)s.heads * d;
  NRS_REQUIRE(ctx, s.ld_x >= row && (!s.y || s.ld_y >= row) && (!bwd || s.ld_g >= row), NRS_ERR_SHAPE,
              "%s: a row of %d heads of %d does not fit its stride (%s)", who, s.heads, d, which);
  NRS_REQUIRE(ctx, (s.y != s.x || s.ld_y == s.ld_x) && (!bwd || s.y != s.g || s.ld_y == s.ld_g), NRS_ERR_ARG,
              "%s: in place needs the same stride (%s)", who, which);
  return NRS_OK;
}

template <bool INTER, bool BWD>
void launch_vec(nrs_ctx* ctx, const Args& a, unsigned grid) {
  switch (lanes_of(a.d)) {
    case 4: NRS_PDL_LAUNCH((head_norm_kernel<4, INTER, BWD>), grid, kThreads, 0, ctx->stream, a); break;
    case 8: NRS_PDL_LAUNCH((head_norm_kernel<8, INTER, BWD>), grid, kThreads, 0, ctx->stream, a); break;
    case 16: NRS_PDL_LAUNCH((head_norm_kernel<16, INTER, BWD>), grid, kThreads, 0, ctx->stream, a); break;
    default: NRS_PDL_LAUNCH((head_norm_kernel<32, INTER, BWD>), grid, kThreads, 0, ctx->stream, a); break;
  }
}

template <bool BWD>
int launch(nrs_ctx* ctx, Args& a, const Shape& sh, float* workspace, int sums /*backward: which sides' dgamma*/) {
  const int st = a.table ? nrs_err_flag(ctx, &a.err) : NRS_OK;
  if (st != NRS_OK) return st;
  bool vec = a.d % 8 == 0 && a.rot % 8 == 0 && a.d <= 256 && ((uintptr_t)a.table & 15) == 0;
  for (Side& s : a.side) {
    if (s.heads == 0) continue;
    vec = vec && (((uintptr_t)s.x | (uintptr_t)s.g | (uintptr_t)s.gamma | (uintptr_t)s.y) & 15) == 0 && s.ld_x % 4 == 0 && s.ld_g % 4 == 0 && s.ld_y % 4 == 0;
  }
  for (Side& s : a.side) {
    vec = vec && (long)a.tokens * s.heads <= 0x3fffffffL;
    s.div = NrsFastDiv(s.heads > 0 ? s.heads : 1);
  }
  a.div_seq = NrsFastDiv(a.seq > 0 ? a.seq : 1);
  plan_blocks(ctx, &a, vec ? kWarps * (32 / lanes_of(a.d)) * kDeep : kWarps, BWD ? kBlocksBwd : kBlocksFwd);
  const unsigned grid = (unsigned)(a.side[0].blocks + a.side[1].blocks);
  if (grid == 0) return NRS_OK;
  if (BWD) {
    if (sums & 1) a.side[0].partial = workspace;
    if (sums & 2) a.side[1].partial = workspace + (size_t)a.side[0].blocks * a.d;
  }
  if (vec) {
    if (sh.interleaved) launch_vec<true, BWD>(ctx, a, grid);
    else launch_vec<false, BWD>(ctx, a, grid);
  } else {
    const size_t smem = BWD ? (size_t)kWarps * a.d * sizeof(float) : 0;   // at most 32 KB
    NRS_PDL_LAUNCH((head_norm_any_kernel<BWD>), grid, kThreads, smem, ctx->stream, a, sh.interleaved);
  }
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

}  // namespace

extern "C" {

int nrs_rotary_table(nrs_ctx* ctx, float* table, int max_len, int rot_dim, float base) {
  NRS_REQUIRE_CTX(ctx);
  NRS_REQUIRE(ctx, max_len >= 0 && rot_dim > 0 && rot_dim % 2 == 0, NRS_ERR_SHAPE, "nrs_rotary_table: %d positions, %d features", max_len, rot_dim);
  NRS_REQUIRE(ctx, base > 0.0f, NRS_ERR_ARG, "nrs_rotary_table: base must be positive");
  if (max_len == 0) return NRS_OK;
  NRS_REQUIRE(ctx, table, NRS_ERR_ARG, "nrs_rotary_table: null table");
  NrsDeviceGuard on(ctx);
  const size_t want = ((size_t)max_len * (rot_dim / 2) + 255) / 256, cap = (size_t)ctx->sm_count * 8;
  NRS_PDL_LAUNCH(rotary_table_kernel, (unsigned)(want < cap ? want : cap), 256, 0, ctx->stream, table, max_len, rot_dim / 2, (double)base);
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

int nrs_qk_norm_rotary_fwd(nrs_ctx* ctx, const float* q, int64_t ld_q, const float* k, int64_t ld_k, const float* gamma_q, const float* gamma_k,
                           const float* table, const int32_t* positions, float* q_out, int64_t ld_q_out, float* k_out, int64_t ld_k_out,
                           int tokens, int seq, int heads_q, int heads_k, int d_head, int rot_dim, int max_len, int interleaved, float eps) {
  NRS_REQUIRE_CTX(ctx);
  const Shape sh{tokens, seq, heads_q, heads_k, d_head, rot_dim, max_len, interleaved != 0, eps};
  int st = check_shape(ctx, __func__, sh, table, positions);
  if (st != NRS_OK) return st;
  Args a{};
  a.side[0] = Side{q, nullptr, gamma_q, q_out, nullptr, (long)ld_q, 0, (long)ld_q_out, heads_q, 0, 0, {}};
  a.side[1] = Side{k, nullptr, gamma_k, k_out, nullptr, (long)ld_k, 0, (long)ld_k_out, heads_k, 0, 0, {}};
  if (tokens == 0) return NRS_OK;
  st = check_side(ctx, __func__, "queries", a.side[0], d_head, false);
  if (st == NRS_OK) st = check_side(ctx, __func__, "keys", a.side[1], d_head, false);
  if (st != NRS_OK) return st;
  a.table = table; a.pos = positions;
  a.tokens = tokens; a.seq = seq; a.d = d_head; a.rot = rot_dim; a.max_len = max_len;
  a.eps = eps; a.inv_d = 1.0f / (float)d_head;
  NrsDeviceGuard on(ctx);
  return launch<false>(ctx, a, sh, nullptr, 0);
}

// (Partial rows of d_head sums: one a block, of which there are as many as the rows fill and at most kBlocksBwd an SM.)
size_t nrs_qk_norm_rotary_workspace(int tokens, int heads_q, int heads_k, int d_head) {
  if (tokens <= 0 || heads_q < 0 || heads_k < 0 || d_head <= 0) return 0;
  constexpr long kMost = 256L * kBlocksBwd + 2;
  const long rows = (long)tokens * ((long)heads_q + heads_k) / kWarps + 2;
  return (size_t)(rows < kMost ? rows : kMost) * d_head * sizeof(float);
}

int nrs_qk_norm_rotary_bwd(nrs_ctx* ctx, const float* g_q, int64_t ld_gq, const float* g_k, int64_t ld_gk, const float* q, int64_t ld_q,
                           const float* k, int64_t ld_k, const float* gamma_q, const float* gamma_k, const float* table,
                           const int32_t* positions, float* dq, int64_t ld_dq, float* dk, int64_t ld_dk, float* dgamma_q, float* dgamma_k,
                           int tokens, int seq, int heads_q, int heads_k, int d_head, int rot_dim, int max_len, int interleaved, float eps,
                           int accumulate, int accumulate_params, void* workspace, size_t workspace_bytes) {
  NRS_REQUIRE_CTX(ctx);
  const Shape sh{tokens, seq, heads_q, heads_k, d_head, rot_dim, max_len, interleaved != 0, eps};
  int st = check_shape(ctx, __func__, sh, table, positions);
  if (st != NRS_OK) return st;
  Args a{};
  a.side[0] = Side{q, g_q, gamma_q, dq, nullptr, (long)ld_q, (long)ld_gq, (long)ld_dq, heads_q, 0, 0, {}};
  a.side[1] = Side{k, g_k, gamma_k, dk, nullptr, (long)ld_k, (long)ld_gk, (long)ld_dk, heads_k, 0, 0, {}};
  if (tokens > 0) {
    st = check_side(ctx, __func__, "queries", a.side[0], d_head, true);
    if (st == NRS_OK) st = check_side(ctx, __func__, "keys", a.side[1], d_head, true);
    if (st != NRS_OK) return st;
    for (const Side& s : a.side)
      NRS_REQUIRE(ctx, !accumulate || !s.heads || !s.y || (s.y != s.g && s.y != s.x), NRS_ERR_ARG, "%s: in place and accumulating at once", __func__);
    const size_t need = nrs_qk_norm_rotary_workspace(tokens, heads_q, heads_k, d_head);
    NRS_REQUIRE(ctx, workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, NRS_ERR_ARG,
                "%s: needs a workspace of %zu bytes on a 16-byte boundary", __func__, need);
  }
  a.table = table; a.pos = positions;
  a.tokens = tokens; a.seq = seq; a.d = d_head; a.rot = rot_dim; a.max_len = max_len;
  a.eps = eps; a.inv_d = 1.0f / (float)d_head; a.accumulate = accumulate != 0;
  NrsDeviceGuard on(ctx);
  if (tokens > 0) {
    st = launch<true>(ctx, a, sh, (float*)workspace, (dgamma_q ? 1 : 0) | (dgamma_k ? 2 : 0));
    if (st != NRS_OK) return st;
  }
  if ((!dgamma_q && !dgamma_k) || (accumulate_params && a.side[0].blocks + a.side[1].blocks == 0)) return NRS_OK;
  NRS_PDL_LAUNCH(head_norm_fold_kernel, dim3((d_head + 31) / 32, 2), 1024, 0, ctx->stream, (const float*)a.side[0].partial, a.side[0].blocks, dgamma_q,
                 (const float*)a.side[1].partial, a.side[1].blocks, dgamma_k, d_head, accumulate_params != 0);
  NRS_LAUNCHED(ctx);
  return NRS_OK;
}

}  // extern "C"
