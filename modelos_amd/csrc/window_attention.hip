// Causal attention through a sliding window, with a few first tokens that stay
// visible (sinks), over padded batches: forward and backward.
//
// Key j is visible to the query at position p of a sequence of tokens
// [start, end) if start <= j <= p < end and (p - j < window or j - start < sinks).
//   o_p = sum_j P_pj v_j,  P_pj = exp(scale q_p.k_j - lse_p),  lse_p = log sum_j exp(scale q_p.k_j)
//   dV = P^T dO,  dS = P (dO V^T - delta),  delta_p = dO_p.o_p,  dQ = scale dS K,  dK = scale dS^T Q
// Positions inside the kernels are relative to the sequence's start.
#include <algorithm>

#include "attn_common.h"

namespace pkm {
namespace {

constexpr int kThreads = 256;  // 4 waves
constexpr int kTile = 64;      // rows of an LDS tile

struct AttnArgs {
  Heads q, k, v, o, dO, dq, dk, dv;
  Heads rest;    // what the rounding left of o at positions [0, rest_rows) of the sequences, or nothing
  float* lse;    // [batch, q_heads, tokens], in units of log2; +inf where nothing is visible
  float* delta;  // [batch, q_heads, tokens]
  const int* starts;
  const int* ends;
  int batch, q_heads, kv_heads, tokens;
  int window, sinks;  // window in [1, tokens] (tokens: no window), sinks in [0, tokens]
  int rest_rows;
  int pack;           // query heads of one key head that share a workgroup: 1, 2 or 4
  // the backward of the sinks from queries past their windows, when it has workgroups of its own
  float* far;  // [pairs, 32-sink blocks, far_chunks, 2 (dK, dV), 32, dim]
  int far_chunks, far_units, dim;  // chunks (0: none), steps of 32 queries in a chunk
  float scale;
};

struct Span {
  int start, n;  // first token and number of tokens of a sequence, inside [0, tokens)
};
__device__ __forceinline__ Span sequence(const AttnArgs& a, int b) {
  const int s = a.starts ? min(max(a.starts[b], 0), a.tokens) : 0;
  const int e = a.ends ? min(max(a.ends[b], 0), a.tokens) : a.tokens;
  return {s, max(e - s, 0)};
}

// Of the pairs (queries p0 .. p1, keys j0 .. j1): are any visible, are all.
__device__ __forceinline__ bool any_visible(int p0, int p1, int j0, int j1, int W, int S) {
  return j0 <= p1 && (p0 - j1 < W || j0 < S);
}
__device__ __forceinline__ bool all_visible(int p0, int p1, int j0, int j1, int W, int S) {
  return j1 <= p0 && (p1 - j0 < W || j1 < S);
}
__device__ __forceinline__ bool visible(int p, int j, int W, int S) { return j <= p && (p - j < W || j < S); }
// The query at position p sees one key alone. Its weight is 1 whatever q and the key are, so their gradients are 0, which
// dS is only up to rounding: dO V^T and delta are summed in different orders.
__device__ __forceinline__ bool lone(int p, int W, int S) { return p == 0 || (W == 1 && S == 0); }

// The key tiles that queries [p0, p1] see: tiles [0, sink) hold the sinks, then those of the window follow.
struct KeyTiles {
  int sink, near, count;
  __device__ __forceinline__ KeyTiles(int p0, int p1, int W, int S) {
    if (p1 < p0) {
      sink = near = count = 0;
      return;
    }
    const int last = p1 / kTile + 1, lo = max(0, p0 - W + 1) / kTile;
    sink = min((min(S, p1 + 1) + kTile - 1) / kTile, lo);
    near = lo - sink;
    count = sink + last - lo;
  }
  __device__ __forceinline__ int tile(int i) const { return i < sink ? i : i + near; }
};

// The steps of 32 queries past the window of the sinks [32 block, 32 block + 32) of a sequence of n tokens, head after head.
struct FarPlan {
  int tile0, tiles, units, used;  // first tile, tiles of a head, steps, chunks that hold any
  int64_t slot;
  __device__ __forceinline__ FarPlan(const AttnArgs& a, int pair, int block, int n) {
    const int p0 = 32 * block + a.window;
    tile0 = p0 / 32;
    tiles = p0 < n ? (n - 1) / 32 + 1 - tile0 : 0;
    units = tiles * (a.q_heads / a.kv_heads);
    used = (units + a.far_units - 1) / a.far_units;
    slot = ((int64_t)pair * ((a.sinks + 31) / 32) + block) * a.far_chunks;
  }
  __device__ __forceinline__ float* part(const AttnArgs& a, int chunk) const {
    return a.far + (slot + chunk) * (2 * 32 * a.dim);
  }
};

// dS as f16. f16 holds numbers from 2^-14 to 2^16 in full, and dS, a gradient times a weight of 1 / keys or so, lies anywhere:
// it is multiplied by a power of two of its column (a query in dQ, a key in dK), the same in both half waves, which
// starts high and falls when a step's largest number reaches 2^15, to bring that below 2^10. Sums are kept in the same
// units. 4096 tokens with gradients of 2^-12: errors of dQ and dK 1.01 and 1.03 times those of rounded results (without it
// 4.6 and 5.7, and NaN where |dS| reaches 2^16). It costs 2 to 4 % of a step of 4 x 4096 tokens, 16 / 8 heads of 128, window 1024
// (0.76 to 0.77 and 0.79 ms), and of 3 x 1777 tokens, 12 heads of 64, dQ 48 to 52 us, dK and dV 48 to 53. For dK and dV the weights
// are taken times 2^kWeightLift, for the same reason. bf16 has float32's range.
template <typename T>
constexpr bool kLifts = __is_same(T, f16_t);
template <typename T>
constexpr int kWeightLift = kLifts<T> ? 12 : 0;

// After a step's numbers: rescale(change) where any of the wave's columns have grown too large, with the exponent to add to that
// of the lane's power of two: less than 0 there, 0 elsewhere.
template <typename F>
__device__ __forceinline__ void lower_lift(const f32x16_t& x, F rescale) {
  float top = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
  if (!__any(top >= 32768.f)) return;
  top = fmaxf(top, swap_halves(top));
  rescale(top >= 32768.f ? min(10 - __builtin_amdgcn_frexp_expf(top), 0) : 0);  // (the exponent of infinity reads as 0)
}

// A workgroup's share of the queries: 4 waves of 32 rows each, `pack` heads of one key head beside each other.
struct QueryBlock {
  int b, kv, head, row;  // the wave's head and its first row
  int first, rows;       // the workgroup's rows
  __device__ __forceinline__ QueryBlock(const AttnArgs& a, int id, int wave) {
    const int pairs = a.batch * a.kv_heads, parts = a.q_heads / a.kv_heads / a.pack;
    const int pair = id % pairs;
    id /= pairs;
    const int part = id % parts;
    id /= parts;
    rows = 128 / a.pack;
    const int blocks = (a.tokens + rows - 1) / rows;
    b = pair / a.kv_heads;
    kv = pair % a.kv_heads;
    head = (kv * parts + part) * a.pack + wave % a.pack;
    first = (blocks - 1 - id) * rows;  // the longest pasts first
    row = first + 32 * (wave / a.pack);
  }
};

// ---------------------------------------------------------------------------
// Forward: S^T = K Q^T per wave of 32 queries and tile of 64 keys, so that a
// lane holds one query's weights: maximum and sum need one exchange between the
// half waves, the weights none before O^T = V^T P^T. One pass over the keys; the weights
// are rounded to the tensors' type for the product, below 2^8 of the row's reference.
// Query heads that share a key head share its tiles in a workgroup, which also keeps
// the queries' span, and with it the tiles at the window's ends, short.
//
// Two workgroups of 4 waves a CU (225 registers; 64 KB of LDS each, two stages). 32768
// tokens, 32 / 8 heads of 128, window 4096: 1.97 to 2.13 ms, 1000 TFLOP/s of visible pairs, 70 % of a
// large matrix product's rate. The matrix cores are busy 55 % of the cycles and the vector units 55 %, at
// a clock that the load pulls to 1.9 GHz; each operand fragment read from LDS feeds one
// product, which is as much as LDS gives (128 bytes a cycle). Measured on the way: tiles through
// registers 2.43 ms, straight to LDS 2.20, reads issued 2 to 3 products ahead 2.08.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void window_fwd_kernel(const AttnArgs a) {
  constexpr int KS = D / 16, DT = D / 32, TB = kTile * D * 2;
  __shared__ __align__(256) uint8_t smem[2 * 2 * TB];
  lds_u8* const lds = (lds_u8*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = lane & 31, h = lane >> 5;
  const QueryBlock qb(a, blockIdx.x, wave);
  const Span seq = sequence(a, qb.b);
  const int W = a.window, S = a.sinks;

  const int row = qb.row + l;
  const int p = row - seq.start;  // the lane's position
  const bool live = row < a.tokens && p >= 0 && p < seq.n;
  const int p0 = max(qb.row - seq.start, 0), p1 = min(qb.row + 31 - seq.start, seq.n - 1);  // the wave's
  const KeyTiles tiles(max(qb.first - seq.start, 0), min(qb.first + qb.rows - 1 - seq.start, seq.n - 1), W, S);

  frag_t q[KS];
  const uint8_t* qrow = live ? a.q.at(qb.b, qb.head, row) : nullptr;
#pragma unroll
  for (int s = 0; s < KS; ++s) q[s] = frag_global<D>(qrow, s, lane);

  const uint8_t* kbase = a.k.at(qb.b, qb.kv, seq.start);
  const uint8_t* vbase = a.v.at(qb.b, qb.kv, seq.start);
  const uint32_t kstride = (uint32_t)(2 * a.k.token), vstride = (uint32_t)(2 * a.v.token);
  const TileLoad<D, kTile> tl(tid);

  f32x16_t o[DT] = {};
  float m = -INFINITY, sum = 0.f;
  const float c = a.scale * 1.44269504f;

  if (tiles.count > 0) {
    const int t0 = tiles.tile(0) * kTile;
    tl.load(lds, kbase + (int64_t)t0 * kstride, kstride, seq.n - t0, tid);
    tl.load(lds + TB, vbase + (int64_t)t0 * vstride, vstride, seq.n - t0, tid);
  }
  tile_wait();
  __syncthreads();
  for (int it = 0; it < tiles.count; ++it) {
    const int j0 = tiles.tile(it) * kTile;
    const uint32_t tile = lds_address(lds) + (it & 1) * 2 * TB;
    const uint32_t krows = tile + rows_at<D>(lane), vcols = tile + TB + cols_at<D>(lane);
    if (it + 1 < tiles.count) {
      const int t1 = tiles.tile(it + 1) * kTile;
      lds_u8* next = lds + ((it + 1) & 1) * 2 * TB;
      tl.load(next, kbase + (int64_t)t1 * kstride, kstride, seq.n - t1, tid);
      tl.load(next + TB, vbase + (int64_t)t1 * vstride, vstride, seq.n - t1, tid);
    }
    if (p0 <= p1 && any_visible(p0, p1, j0, j0 + kTile - 1, W, S)) {
      f32x16_t s[2] = {};
      frag_t f0[3], f1[3];
      const auto rows = [&](int i) {
        f0[i % 3] = frag_rows<D>(krows, 0, i);
        f1[i % 3] = frag_rows<D>(krows, 32, i);
      };
      rows(0);
      rows(1);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        if (i + 2 < KS) rows(i + 2);
        keep_order();
        s[0] = mfma32<T>(f0[i % 3], q[i], s[0]);
        s[1] = mfma32<T>(f1[i % 3], q[i], s[1]);
        keep_order();
      }
      frag_t fv[4];
      const auto cols = [&](int i) { fv[i % 4] = frag_cols<D>(vcols, 16 * (i / DT), i % DT); };
      cols(0);
      cols(1);
      cols(2);
      if (!all_visible(p0, p1, j0, j0 + kTile - 1, W, S)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = j0 + 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3);
            s[kb][i] = visible(p, j, W, S) ? s[kb][i] : -INFINITY;
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
      top = fmaxf(top, fmaxf(swap_halves(top), m));
      // the reference moves only when a row's largest logit has grown by more than 8 in log2 (weights stay below 2^8;
      // half of the tiles of a long row would otherwise rescale 64 numbers a lane)
      if (__any((top - m) * c > 8.f)) {
        const float f = m == -INFINITY ? 0.f : exp2_raw((m - top) * c);
        sum *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[t][i] *= f;
        m = top;
      }
      const float mc = m == -INFINITY ? 0.f : m * c;
      frag_t pf[4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[kb][i] = exp2_raw(__builtin_fmaf(s[kb][i], c, -mc));
          sum += s[kb][i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) pf[2 * kb + i / 4][i % 4] = pack2<T>(s[kb][2 * i], s[kb][2 * i + 1]);
      }
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) {
        if (i + 3 < 4 * DT) cols(i + 3);
        keep_order();
        o[i % DT] = mfma32<T>(fv[i % 4], pf[i / DT], o[i % DT]);
        keep_order();
      }
    }
    tile_wait();
    __syncthreads();
  }

  if (row >= a.tokens) return;
  sum += swap_halves(sum);
  const bool some = live && sum != 0.f;  // NaN counts as something
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = some ? o[t][i] : 0.f;
  store_row<T, D>(a.o.at(qb.b, qb.head, row), o, some ? 1.f / sum : 0.f, lane,
                  a.rest.p && live && p < a.rest_rows ? a.rest.at(qb.b, qb.head, p) : nullptr);
  if (a.lse && h == 0) {
    a.lse[((int64_t)qb.b * a.q_heads + qb.head) * a.tokens + row] =
        some ? m * c + __builtin_amdgcn_logf(sum) : INFINITY;
  }
}

// ---------------------------------------------------------------------------
// Backward, dQ: as the forward, dS^T = P^T (V dO^T - delta), dQ^T = K^T dS^T. The 4 x 4096 tokens of a training
// step (16 / 8 heads of 128, window 1024): 0.25 to 0.28 ms, matrix cores 49 %, vector units 43 % of the cycles.
//
// delta comes from the output, with what its rounding left where that was kept: for rows that see few keys, which are
// all of a short window's and the first of every sequence. What an error in it puts into a row's dS
// adds up to sum_j dS_j (which is 0), so the sum corrects the delta that dK reads. dS enters its
// product as two 16-bit numbers, itself rounded and the rest: keys have a common part,
// which the exact dS, whose sum is 0, cancels and the roundings of one would not (relative error
// of dQ 2.7e-3 with one, 2.0e-3 with two in bf16, where the result's own rounding is 1.7e-3).
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void window_dq_kernel(const AttnArgs a) {
  constexpr int KS = D / 16, DT = D / 32, TB = kTile * D * 2;
  __shared__ __align__(256) uint8_t smem[2 * 2 * TB];
  lds_u8* const lds = (lds_u8*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = lane & 31, h = lane >> 5;
  const QueryBlock qb(a, blockIdx.x, wave);
  const Span seq = sequence(a, qb.b);
  const int W = a.window, S = a.sinks;
  const int row = qb.row + l;
  const int p = row - seq.start;
  const bool live = row < a.tokens && p >= 0 && p < seq.n;
  const int p0 = max(qb.row - seq.start, 0), p1 = min(qb.row + 31 - seq.start, seq.n - 1);
  const KeyTiles tiles(max(qb.first - seq.start, 0), min(qb.first + qb.rows - 1 - seq.start, seq.n - 1), W, S);

  frag_t q[KS], g[KS];
  const uint8_t* qrow = live ? a.q.at(qb.b, qb.head, row) : nullptr;
  const uint8_t* grow = live ? a.dO.at(qb.b, qb.head, row) : nullptr;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    q[s] = frag_global<D>(qrow, s, lane);
    g[s] = frag_global<D>(grow, s, lane);
  }
  const int64_t at = ((int64_t)qb.b * a.q_heads + qb.head) * a.tokens + row;
  float lse = live ? a.lse[at] : INFINITY;
  float delta = 0.f, sum = 0.f;
  // dS and its sums are in units of 2^-lift, by way of lse; 2^80 times the largest dS of f16 inputs fits float32
  int lift = kLifts<T> ? 80 : 0;
  lse -= (float)lift;
  const uint8_t* orow = live ? a.o.at(qb.b, qb.head, row) : nullptr;
#pragma unroll
  for (int s = 0; s < KS; ++s)
    delta = vec_dot<T>(__builtin_bit_cast(uint4, frag_global<D>(orow, s, lane)), __builtin_bit_cast(uint4, g[s]), delta);
  if (a.rest.p && p0 < a.rest_rows) {
    const uint8_t* rrow = live && p < a.rest_rows ? a.rest.at(qb.b, qb.head, p) : nullptr;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      delta = vec_dot<T>(__builtin_bit_cast(uint4, frag_global<D>(rrow, s, lane)), __builtin_bit_cast(uint4, g[s]), delta);
  }
  delta += swap_halves(delta);

  const uint8_t* kbase = a.k.at(qb.b, qb.kv, seq.start);
  const uint8_t* vbase = a.v.at(qb.b, qb.kv, seq.start);
  const uint32_t kstride = (uint32_t)(2 * a.k.token), vstride = (uint32_t)(2 * a.v.token);
  const TileLoad<D, kTile> tl(tid);
  f32x16_t dq[DT] = {};
  const float c = a.scale * 1.44269504f;

  if (tiles.count > 0) {
    const int t0 = tiles.tile(0) * kTile;
    tl.load(lds, kbase + (int64_t)t0 * kstride, kstride, seq.n - t0, tid);
    tl.load(lds + TB, vbase + (int64_t)t0 * vstride, vstride, seq.n - t0, tid);
  }
  tile_wait();
  __syncthreads();
  for (int it = 0; it < tiles.count; ++it) {
    const int j0 = tiles.tile(it) * kTile;
    const uint32_t tile = lds_address(lds) + (it & 1) * 2 * TB;
    const uint32_t krows = tile + rows_at<D>(lane), vrows = krows + TB, kcols = tile + cols_at<D>(lane);
    if (it + 1 < tiles.count) {
      const int t1 = tiles.tile(it + 1) * kTile;
      lds_u8* next = lds + ((it + 1) & 1) * 2 * TB;
      tl.load(next, kbase + (int64_t)t1 * kstride, kstride, seq.n - t1, tid);
      tl.load(next + TB, vbase + (int64_t)t1 * vstride, vstride, seq.n - t1, tid);
    }
    if (p0 <= p1) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int ja = j0 + 32 * kb;
        if (!any_visible(p0, p1, ja, ja + 31, W, S)) continue;
        f32x16_t s = {}, dp = {};
        frag_t fk[3], fv[3];
        const auto rows = [&](int i) {
          fk[i % 3] = frag_rows<D>(krows, 32 * kb, i);
          fv[i % 3] = frag_rows<D>(vrows, 32 * kb, i);
        };
        rows(0);
        rows(1);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          if (i + 2 < KS) rows(i + 2);
          keep_order();
          s = mfma32<T>(fk[i % 3], q[i], s);
          dp = mfma32<T>(fv[i % 3], g[i], dp);
          keep_order();
        }
        const auto cols = [&](int i) { fk[i % 3] = frag_cols<D>(kcols, 32 * kb + 16 * (i / DT), i % DT); };
        cols(0);
        cols(1);
        if (!all_visible(p0, p1, ja, ja + 31, W, S)) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[i] = visible(p, ja + 8 * (i >> 2) + 4 * h + (i & 3), W, S) ? s[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = exp2_raw(__builtin_fmaf(s[i], c, -lse)) * (dp[i] - delta);
          sum += s[i];
        }
        if constexpr (kLifts<T>) {
          lower_lift(s, [&](int change) {
            const float f = ldexpf(1.f, change);
            lift += change;
            lse -= (float)change;
            sum *= f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] *= f;
#pragma unroll
            for (int t = 0; t < DT; ++t) dq[t] *= f;
          });
        }
        frag_t f[2], r[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[8 * i + 2 * e], y = s[8 * i + 2 * e + 1];
            f[i][e] = pack2<T>(x, y);
            r[i][e] = pack2<T>(x - unpack1<T>(f[i][e] & 0xffffu), y - unpack1<T>(f[i][e] >> 16));
          }
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) {
          if (i + 2 < 2 * DT) cols(i + 2);
          keep_order();
          dq[i % DT] = mfma32<T>(fk[i % 3], f[i / DT], dq[i % DT]);
          dq[i % DT] = mfma32<T>(fk[i % 3], r[i / DT], dq[i % DT]);
          keep_order();
        }
      }
    }
    tile_wait();
    __syncthreads();
  }
  sum = ldexpf(sum + swap_halves(sum), -lift);
  if (row >= a.tokens) return;
  if (live && h == 0) a.delta[at] = delta + sum;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[t][i] = live ? dq[t][i] : 0.f;
  store_row<T, D>(a.dq.at(qb.b, qb.head, row), dq, lone(p, W, S) ? 0.f : ldexpf(a.scale, -lift), lane);
}

// ---------------------------------------------------------------------------
// Backward, dK and dV: 128 keys a workgroup; the tiles hold 64 queries and
// their dO, of every query head of the key head in turn (a shared head's
// gradient is summed in registers, in a fixed order). Of the 8 waves, 4 take 32
// keys each with the tiles' first 32 queries, 4 the same with the second. The keys stay in LDS and the
// values in registers: with both in registers a wave needs more than the 256
// that let two waves share a SIMD. Three stages of tiles, two of them on their way.
//
// The same step: 0.33 to 0.38 ms (one wave a SIMD 0.42). Matrix cores 34 %, vector units 32 %: a wave
// issues a third of its time, waits a third for the matrix core and a third for LDS and the barrier.
// Copies of the kernel without its exponentials, either pair of products, its LDS reads or its loads took
// 0.30 to 0.33 ms each, so no one of them is the limit; the two halves half a step apart,
// with a second barrier, took 0.36 to 0.39, priorities for either half changed nothing.
// ---------------------------------------------------------------------------
constexpr int kQueries = 32;
template <int D>
struct DkvLds {
  static constexpr int TB = kQueries * D * 2, BUF = 2 * TB + 2 * kQueries * 4;  // a step's
};

// One step: 32 queries, their dO, lse and delta, and the wave's 32 keys in LDS, their values v.
// masked(i): the row i of the lane's column is not visible; all: none is masked. lone0: the step's first query sees one key alone.
// dk and dv are in units that take_units ends; up: the lane's.
template <typename T, int D, typename F>
__device__ __forceinline__ void dkv_step(const lds_u8* qtile, const lds_u8* gtile, const lds_u8* lses,
                                         const lds_u8* deltas, const lds_u8* keys, const frag_t (&v)[D / 16], float c,
                                         bool all, bool lone0, F masked, f32x16_t (&dk)[D / 32], f32x16_t (&dv)[D / 32], float& up,
                                         int lane) {
  constexpr int KS = D / 16, DT = D / 32;
  asm volatile("" : "+v"(lane));  // the addresses below are worked out anew in each step: kept over the loop, they spill
  const int h = lane >> 5;
  const uint32_t at = rows_at<D>(lane), qrows = lds_address(qtile) + at, grows = lds_address(gtile) + at;
  const uint32_t krows = lds_address(keys) + at;
  f32x16_t s = {}, dp = {};
  frag_t fq[3], fk[3], fg[3];
  const auto rows = [&](int i) {
    fq[i % 3] = frag_rows<D>(qrows, 0, i);
    fk[i % 3] = frag_rows<D>(krows, 0, i);
    fg[i % 3] = frag_rows<D>(grows, 0, i);
  };
  rows(0);
  rows(1);
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    if (i + 2 < KS) rows(i + 2);
    keep_order();
    s = mfma32<T>(fq[i % 3], fk[i % 3], s);
    dp = mfma32<T>(fg[i % 3], v[i], dp);
    keep_order();
  }
  const uint32_t qcols = lds_address(qtile) + cols_at<D>(lane), gcols = lds_address(gtile) + cols_at<D>(lane);
  const auto cols = [&](int i) {
    fg[i % 3] = frag_cols<D>(gcols, 16 * (i / DT), i % DT);
    fq[i % 3] = frag_cols<D>(qcols, 16 * (i / DT), i % DT);
  };
  cols(0);
  cols(1);
  if (!all) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = masked(8 * (i >> 2) + 4 * h + (i & 3)) ? -INFINITY : s[i];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x4_t lse = *(const lds_f32x4*)(lses + 4 * (8 * e + 4 * h));
    const f32x4_t delta = *(const lds_f32x4*)(deltas + 4 * (8 * e + 4 * h));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 4 * e + r;
      s[i] = exp2_raw(__builtin_fmaf(s[i], c, (float)kWeightLift<T> - lse[r]));
      dp[i] = s[i] * (dp[i] - delta[r]);
      if constexpr (kLifts<T>) dp[i] *= up;
    }
  }
  if (lone0) dp[0] = h == 0 ? 0.f * dp[0] : dp[0];
  if constexpr (kLifts<T>) {
    lower_lift(dp, [&](int change) {
      const float f = ldexpf(1.f, change);
      up *= f;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] *= f;
#pragma unroll
      for (int t = 0; t < DT; ++t) dk[t] *= f;
    });
  }
  frag_t pf[2], sf[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pf[i][e] = pack2<T>(s[8 * i + 2 * e], s[8 * i + 2 * e + 1]);
      sf[i][e] = pack2<T>(dp[8 * i + 2 * e], dp[8 * i + 2 * e + 1]);
    }
#pragma unroll
  for (int i = 0; i < 2 * DT; ++i) {
    if (i + 2 < 2 * DT) cols(i + 2);
    keep_order();
    dv[i % DT] = mfma32<T>(fg[i % 3], pf[i / DT], dv[i % DT]);
    dk[i % DT] = mfma32<T>(fq[i % 3], sf[i / DT], dk[i % DT]);
    keep_order();
  }
}

constexpr float kUp = 1152921504606846976.f;  // 2^60: what `up` starts from; times 2^12 and the largest f16 dS it fits float32
template <typename T, int DT>
__device__ __forceinline__ void take_units(f32x16_t (&dk)[DT], f32x16_t (&dv)[DT], float up) {
  if constexpr (kLifts<T>) {
    const float v = ldexpf(1.f, -kWeightLift<T>), k = v / up;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      dk[t] *= k;
      dv[t] *= v;
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(512, 2) void window_dkv_kernel(const AttnArgs a) {
  constexpr int KS = D / 16, DT = D / 32, TB = kTile * D * 2, KEYS = 128 * D * 2;
  constexpr int STAGE = 2 * TB + 8 * 256, LOADS = 2 * TileLoad<D, kTile, 8>::N + 1;  // a wave's loads of a stage
  __shared__ __align__(256) uint8_t smem[KEYS + 3 * STAGE];
  lds_u8* const keys = (lds_u8*)smem;
  lds_u8* const lds = keys + KEYS;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = lane & 31, h = lane >> 5, kw = wave & 3, qw = wave >> 2;
  const int pairs = a.batch * a.kv_heads, pair = blockIdx.x % pairs;
  const int b = pair / a.kv_heads, kv = pair % a.kv_heads, G = a.q_heads / a.kv_heads;
  const int first = blockIdx.x / pairs * 128;  // the key block's rows; the first ones are read by most queries
  const Span seq = sequence(a, b);
  const int W = a.window, S = a.far_chunks ? 0 : a.sinks, n = seq.n;
  const int row = first + 32 * kw + l;
  const int key = row - seq.start;
  const bool live = row < a.tokens && key >= 0 && key < n;
  const int k0 = max(first + 32 * kw - seq.start, 0), k1 = min(first + 32 * kw + 31 - seq.start, n - 1);
  // the queries that see the block: from its first key to the window's end of its last, or all of them
  const int b0 = max(first - seq.start, 0), b1 = min(first + 127 - seq.start, n - 1);
  int tile0 = 0, count = 0;
  if (b0 <= b1) {
    const int last = b0 < S ? n - 1 : min(n - 1, b1 + W - 1);
    tile0 = b0 / kTile;
    count = last / kTile + 1 - tile0;
  }
  const int total = count * G;

  frag_t v[KS];
  const uint8_t* vrow = live ? a.v.at(b, kv, row) : nullptr;
#pragma unroll
  for (int s = 0; s < KS; ++s) v[s] = frag_global<D>(vrow, s, lane);
  const TileLoad<D, kTile, 8> tl(tid);
  const uint32_t qstride = (uint32_t)(2 * a.q.token), gstride = (uint32_t)(2 * a.dO.token);
  // the next stage to load: its head, first row, place in the ring and addresses
  int load_head = kv * G, load_t0 = tile0 * kTile, load_at = 0;
  const uint8_t *qat, *gat;
  int64_t sat;
  const auto start_head = [&] {
    load_t0 = tile0 * kTile;
    qat = a.q.at(b, load_head, seq.start + load_t0);
    gat = a.dO.at(b, load_head, seq.start + load_t0);
    sat = ((int64_t)b * a.q_heads + load_head) * a.tokens + seq.start + load_t0;
  };
  const auto load = [&] {
    const int t0 = load_t0;
    lds_u8* buf = lds + load_at * STAGE;
    tl.load(buf, qat, qstride, n - t0, tid);
    tl.load(buf + TB, gat, gstride, n - t0, tid);
    // 64 rows' lse by wave 0, delta by wave 1; the other waves load lse too, to where nobody reads it, so that
    // every wave has as many loads in flight
    const float* from = (wave == 1 ? a.delta : a.lse) + sat;
    const u32x4_t rs = {(uint32_t)(uintptr_t)from, (uint32_t)((uintptr_t)from >> 32), 0x7fffffffu, 0x00020000u};
    load_lds4(rs, buf + 2 * TB + 256 * wave, 4 * (uint32_t)min(lane, n - t0 - 1));
    load_at = load_at == 2 ? 0 : load_at + 1;
    load_t0 += kTile;
    qat += (uint64_t)kTile * qstride;
    gat += (uint64_t)kTile * gstride;
    sat += kTile;
    if (load_t0 == (tile0 + count) * kTile) {
      ++load_head;
      start_head();
    }
  };

  f32x16_t dk[DT] = {}, dv[DT] = {};
  float up = kUp;
  const float c = a.scale * 1.44269504f;
  if (total > 0) {
    // rows of the block before the sequence's start are read as they are, those past its end repeat its last: whatever they
    // hold, NaN too, stays in their own columns of the products, which `live` drops
    const TileLoad<D, 128, 8> kl(tid);
    kl.load(keys, a.k.at(b, kv, first), (uint32_t)(2 * a.k.token), seq.start + n - first, tid);
    start_head();
    load();
    if (total > 1) load();
  }
  tile_wait();  // and for v: the compiler does not know of the loads to LDS and would wait for them at its use
  int pa = tile0 * kTile + kQueries * qw, ring = 0;  // the wave's queries, the stage's place
  for (int it = 0; it < total; ++it) {
    // stage it has come, of every wave's loads; stage it - 1 is read no more
    if (it + 1 < total) {
      tile_wait<LOADS>();
    } else {
      tile_wait();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (it + 2 < total) load();
    if (k0 <= k1 && any_visible(pa, pa + kQueries - 1, k0, k1, W, S)) {
      const lds_u8* buf = lds + ring * STAGE;
      dkv_step<T, D>(buf + TB / 2 * qw, buf + TB + TB / 2 * qw, buf + 2 * TB + 128 * qw, buf + 2 * TB + 256 + 128 * qw,
                     keys + 32 * kw * (D * 2), v, c,
                     pa + kQueries <= n && all_visible(pa, pa + kQueries - 1, k0, k1, W, S), pa == 0,
                     [&](int i) { return !(pa + i < n && visible(pa + i, key, W, S)); }, dk, dv, up, lane);
    }
    ring = ring == 2 ? 0 : ring + 1;
    pa += kTile;
    if (pa >= (tile0 + count) * kTile) pa -= count * kTile;
  }
  take_units<T>(dk, dv, up);
  // the two query halves' sums: the waves of the first finish dK, those of the second dV
  __syncthreads();
  static_assert(8 * 32 * D * 4 <= KEYS + 3 * STAGE, "eight waves' sums fit");
  float* const sums = (float*)smem + lane;
  const auto give = [&](const f32x16_t(&x)[DT], int slot) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[slot * (32 * D) + (t * 16 + i) * 64] = x[t][i];
  };
  const auto finish = [&](f32x16_t(&x)[DT], int slot, const Heads& to, float f, int part) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[t][i] += sums[slot * (32 * D) + (t * 16 + i) * 64];
    if (a.far_chunks && live && key < a.sinks) {  // the far queries' part, in their order
      const FarPlan far(a, pair, key / 32, n);
      for (int i = 0; i < far.used; ++i) {
        const float* from = far.part(a, i) + part + (int64_t)(key % 32) * D + 4 * h;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4_t y = *(const f32x4_t*)(from + 32 * t + 8 * e);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[t][4 * e + r] += y[r];
          }
      }
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[t][i] = live ? x[t][i] : 0.f;
    store_row<T, D>(to.at(b, kv, row), x, f, lane);
  };
  if (qw == 0) {
    give(dv, 4 + kw);
  } else {
    give(dk, kw);
  }
  __syncthreads();
  if (row >= a.tokens) return;
  if (qw == 0) {
    finish(dk, kw, a.dk, W == 1 && a.sinks == 0 ? 0.f : a.scale, 0);
  } else {
    finish(dv, 4 + kw, a.dv, 1.f, 32 * D);
  }
}

// The sinks' gradients from the queries past their windows: few keys, most queries. A workgroup takes 32 sinks and
// a chunk of those queries' steps, four at a time, one a wave; its sums go to the workspace in float32 for
// window_dkv_kernel. Left in the first key block's workgroup, these steps were the kernel's longest path: 585 us
// against 335 without sinks at 4096 tokens, window 1024.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void window_far_kernel(const AttnArgs a) {
  constexpr int KS = D / 16, DT = D / 32, TB = DkvLds<D>::TB, BUF = DkvLds<D>::BUF, KEYS = 32 * D * 2;
  __shared__ __align__(256) uint8_t smem[KEYS + 4 * BUF];
  lds_u8* const keys = (lds_u8*)smem;
  lds_u8* const lds = keys + KEYS;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = lane & 31, h = lane >> 5;
  const int pairs = a.batch * a.kv_heads, pair = blockIdx.x % pairs;
  const int chunk = blockIdx.x / pairs % a.far_chunks, block = blockIdx.x / pairs / a.far_chunks;
  const int b = pair / a.kv_heads, kv = pair % a.kv_heads, G = a.q_heads / a.kv_heads;
  const Span seq = sequence(a, b);
  const int W = a.window, n = seq.n, S = min(a.sinks, n);
  const FarPlan far(a, pair, block, n);
  if (chunk >= far.used) return;
  const int key = 32 * block + l;

  frag_t v[KS];
  const uint8_t* vrow = key < S ? a.v.at(b, kv, seq.start + key) : nullptr;
#pragma unroll
  for (int s = 0; s < KS; ++s) v[s] = frag_global<D>(vrow, s, lane);
  const TileLoad<D, 32> tl(tid);
  tl.load(keys, a.k.at(b, kv, seq.start + 32 * block), (uint32_t)(2 * a.k.token), S - 32 * block, tid);
  f32x16_t dk[DT] = {}, dv[DT] = {};
  float up = kUp;
  const float c = a.scale * 1.44269504f;
  const int end = min((chunk + 1) * a.far_units, far.units);
  for (int u0 = chunk * a.far_units; u0 < end; u0 += 4) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int u = min(u0 + w, end - 1), head = kv * G + u / far.tiles, t0 = (far.tile0 + u % far.tiles) * kQueries;
      lds_u8* buf = lds + w * BUF;
      tl.load(buf, a.q.at(b, head, seq.start + t0), (uint32_t)(2 * a.q.token), n - t0, tid);
      tl.load(buf + TB, a.dO.at(b, head, seq.start + t0), (uint32_t)(2 * a.dO.token), n - t0, tid);
    }
    const int u = min(u0 + wave, end - 1), head = kv * G + u / far.tiles, t0 = (far.tile0 + u % far.tiles) * kQueries;
    const float* from = h ? a.delta : a.lse;
    const float stat =
        t0 + l < n ? from[((int64_t)b * a.q_heads + head) * a.tokens + seq.start + t0 + l] : (h ? 0.f : INFINITY);
    *(__attribute__((address_space(3))) float*)(lds + wave * BUF + 2 * TB + 4 * lane) = stat;
    tile_wait();
    __syncthreads();
    if (u0 + wave < end) {
      const lds_u8* buf = lds + wave * BUF;
      dkv_step<T, D>(buf, buf + TB, buf + 2 * TB, buf + 2 * TB + 4 * kQueries, keys, v, c,
                     t0 - (32 * block + 31) >= W && 32 * block + 31 < S, false,
                     [&](int i) { return t0 + i - key < W || key >= S; }, dk, dv, up, lane);
    }
    __syncthreads();
  }
  take_units<T>(dk, dv, up);
  // the waves' sums: 2 and 3 go to 0 and 1, then 1 to 0
  float* const sums = (float*)smem;
  static_assert(4 * 32 * D * 4 <= KEYS + 4 * BUF, "two waves' sums fit");
#pragma unroll
  for (int half = 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sums[(((wave - half) * 2 * DT + t) * 16 + i) * 64 + lane] = dk[t][i];
          sums[(((wave - half) * 2 * DT + DT + t) * 16 + i) * 64 + lane] = dv[t][i];
        }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          dk[t][i] += sums[((wave * 2 * DT + t) * 16 + i) * 64 + lane];
          dv[t][i] += sums[((wave * 2 * DT + DT + t) * 16 + i) * 64 + lane];
        }
    }
    __syncthreads();
  }
  if (wave != 0) return;
  float* to = far.part(a, chunk) + (int64_t)l * D + 4 * h;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      *(f32x4_t*)(to + 32 * t + 8 * e) = (f32x4_t){dk[t][4 * e], dk[t][4 * e + 1], dk[t][4 * e + 2], dk[t][4 * e + 3]};
      *(f32x4_t*)(to + 32 * D + 32 * t + 8 * e) =
          (f32x4_t){dv[t][4 * e], dv[t][4 * e + 1], dv[t][4 * e + 2], dv[t][4 * e + 3]};
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_heads(const char* what, const char* name, const pkm_heads_t* x) {
  PKM_REQUIRE(x != nullptr && x->data != nullptr, PKM_ERR_INVALID_ARGUMENT, "%s: %s is NULL", what, name);
  PKM_REQUIRE(((uintptr_t)x->data & 15) == 0 && x->batch % 8 == 0 && x->head % 8 == 0 && x->token % 8 == 0,
              PKM_ERR_UNSUPPORTED, "%s: %s needs 16-byte aligned data and strides that are multiples of 8", what, name);
  PKM_REQUIRE(x->batch >= 0 && x->head >= 0 && x->token >= 0 && x->token < (1 << 22), PKM_ERR_UNSUPPORTED,
              "%s: %s needs strides >= 0 and a token stride below 2^22", what, name);
  return PKM_OK;
}

Heads heads(const pkm_heads_t* x) { return {(uint8_t*)x->data, x->batch, x->head, x->token}; }

int fill_args(const char* what, AttnArgs* a, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t tokens,
              int64_t dim, int dtype, int64_t window, int64_t sinks, float scale) {
  PKM_REQUIRE(batch >= 0 && tokens >= 0 && q_heads > 0 && kv_heads > 0 && window >= 0 && sinks >= 0,
              PKM_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  PKM_REQUIRE(q_heads % kv_heads == 0, PKM_ERR_INVALID_ARGUMENT, "%s: %lld query heads do not share %lld key heads",
              what, (long long)q_heads, (long long)kv_heads);
  PKM_REQUIRE(scale > 0.f && scale <= 3.0e38f, PKM_ERR_INVALID_ARGUMENT, "%s: scale has to be positive and finite", what);
  PKM_REQUIRE((dim == 64 || dim == 128) && (dtype == PKM_DTYPE_BF16 || dtype == PKM_DTYPE_F16), PKM_ERR_UNSUPPORTED,
              "%s: head dims 64 and 128 in bf16 and f16 are supported", what);
  PKM_REQUIRE(tokens < (1 << 24) && batch < (1 << 24) && q_heads < (1 << 24) && batch * q_heads < (1 << 24) &&
                  batch * q_heads * ((tokens + 31) / 32) < (1ll << 31),
              PKM_ERR_UNSUPPORTED, "%s: too many tokens or heads", what);
  // a launch takes fewer than 2^32 threads: 256 a workgroup, with the far sinks' too, and 512 for dK and dV
  const int64_t share = q_heads / kv_heads, pack = share % 4 == 0 ? 4 : share % 2 == 0 ? 2 : 1, rows = 128 / pack;
  PKM_REQUIRE(batch * (q_heads / pack) * ((tokens + rows - 1) / rows) < (1 << 24) &&
                  batch * kv_heads * ((std::min(sinks, tokens) + 31) / 32) < (1 << 24) &&
                  batch * kv_heads * ((tokens + 127) / 128) < (1 << 23),
              PKM_ERR_UNSUPPORTED, "%s: too many tokens or heads", what);
  a->batch = (int)batch;
  a->q_heads = (int)q_heads;
  a->kv_heads = (int)kv_heads;
  a->tokens = (int)tokens;
  a->window = (int)(window == 0 || window > tokens ? tokens : window);
  a->sinks = (int)(sinks > tokens ? tokens : sinks);
  a->rest_rows = a->window <= PKM_ATTN_REST_TOKENS ? (int)tokens : PKM_ATTN_REST_TOKENS;
  a->scale = scale;
  a->dim = (int)dim;
  a->pack = (int)pack;
  return PKM_OK;
}

unsigned query_blocks(const AttnArgs& a) {
  const int rows = 128 / a.pack;
  return (unsigned)(a.batch * (a.q_heads / a.pack) * ((a.tokens + rows - 1) / rows));
}

// Whether the sinks' far queries get workgroups of their own, and how many: they do where a first key block would
// otherwise take more than twice the steps of the others. 512 workgroups in all, of 16 steps at least.
void plan_far(AttnArgs* a) {
  a->far_chunks = 0;
  if (a->sinks == 0 || a->tokens <= 2 * ((int64_t)a->window + 128)) return;
  const int64_t units = (int64_t)((a->tokens - a->window + 31) / 32 + 1) * (a->q_heads / a->kv_heads);
  const int64_t blocks = (int64_t)a->batch * a->kv_heads * ((a->sinks + 31) / 32);
  const int64_t chunks = blocks >= 512 ? 1 : 512 / blocks;
  int64_t each = (units + chunks - 1) / chunks;
  each = each < 16 ? 16 : (each + 3) / 4 * 4;
  a->far_units = (int)each;
  a->far_chunks = (int)((units + each - 1) / each);
}

int64_t delta_bytes(const AttnArgs& a) {
  return ((int64_t)a.batch * a.q_heads * a.tokens * (int64_t)sizeof(float) + 15) / 16 * 16;
}
int64_t far_bytes(const AttnArgs& a) {
  return (int64_t)a.batch * a.kv_heads * ((a.sinks + 31) / 32) * a.far_chunks * 2 * 32 * a.dim * (int64_t)sizeof(float);
}

template <typename T, int D>
void launch_fwd(const AttnArgs& a, hipStream_t st) {
  window_fwd_kernel<T, D><<<query_blocks(a), kThreads, 0, st>>>(a);
}

template <typename T, int D>
void launch_bwd(const AttnArgs& a, hipStream_t st) {
  window_dq_kernel<T, D><<<query_blocks(a), kThreads, 0, st>>>(a);  // and delta
  if (a.far_chunks) {
    const unsigned grid = (unsigned)(a.batch * a.kv_heads * ((a.sinks + 31) / 32) * a.far_chunks);
    window_far_kernel<T, D><<<grid, kThreads, 0, st>>>(a);
  }
  window_dkv_kernel<T, D><<<(unsigned)(a.batch * a.kv_heads * ((a.tokens + 127) / 128)), 512, 0, st>>>(a);
}

}  // namespace
}  // namespace pkm

using namespace pkm;

extern "C" int pkm_window_attn_fwd(const pkm_heads_t* q, const pkm_heads_t* k, const pkm_heads_t* v,
                                   const int32_t* starts, const int32_t* ends, int64_t batch, int64_t q_heads,
                                   int64_t kv_heads, int64_t tokens, int64_t dim, int dtype, int64_t window,
                                   int64_t sinks, float scale, const pkm_heads_t* out, const pkm_heads_t* rest, float* lse,
                                   void* stream) {
  const char* what = "pkm_window_attn_fwd";
  AttnArgs a = {};
  int rc = fill_args(what, &a, batch, q_heads, kv_heads, tokens, dim, dtype, window, sinks, scale);
  if (rc != PKM_OK) return rc;
  if (batch == 0 || tokens == 0) return PKM_OK;
  if ((rc = check_heads(what, "q", q)) || (rc = check_heads(what, "k", k)) || (rc = check_heads(what, "v", v)) ||
      (rc = check_heads(what, "out", out)) || (rest != nullptr && (rc = check_heads(what, "rest", rest))))
    return rc;
  a.q = heads(q), a.k = heads(k), a.v = heads(v), a.o = heads(out);
  if (rest != nullptr) a.rest = heads(rest);
  a.starts = starts, a.ends = ends, a.lse = lse;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKM_DTYPE_BF16) {
    dim == 128 ? launch_fwd<bf16_t, 128>(a, st) : launch_fwd<bf16_t, 64>(a, st);
  } else {
    dim == 128 ? launch_fwd<f16_t, 128>(a, st) : launch_fwd<f16_t, 64>(a, st);
  }
  return pkm_check_launch(what);
}

extern "C" size_t pkm_window_attn_bwd_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t tokens,
                                                     int64_t dim, int64_t window, int64_t sinks) {
  AttnArgs a = {};
  if (batch <= 0 || tokens <= 0 ||
      fill_args("pkm_window_attn_bwd_workspace_size", &a, batch, q_heads, kv_heads, tokens, dim, PKM_DTYPE_BF16, window,
                sinks, 1.f) != PKM_OK)
    return 0;
  plan_far(&a);
  return (size_t)(delta_bytes(a) + far_bytes(a));
}

extern "C" int pkm_window_attn_bwd(const pkm_heads_t* q, const pkm_heads_t* k, const pkm_heads_t* v,
                                   const pkm_heads_t* out, const pkm_heads_t* rest, const float* lse,
                                   const pkm_heads_t* grad_out,
                                   const int32_t* starts, const int32_t* ends, int64_t batch, int64_t q_heads,
                                   int64_t kv_heads, int64_t tokens, int64_t dim, int dtype, int64_t window,
                                   int64_t sinks, float scale, const pkm_heads_t* dq, const pkm_heads_t* dk,
                                   const pkm_heads_t* dv, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "pkm_window_attn_bwd";
  AttnArgs a = {};
  int rc = fill_args(what, &a, batch, q_heads, kv_heads, tokens, dim, dtype, window, sinks, scale);
  if (rc != PKM_OK) return rc;
  if (batch == 0 || tokens == 0) return PKM_OK;
  if ((rc = check_heads(what, "q", q)) || (rc = check_heads(what, "k", k)) || (rc = check_heads(what, "v", v)) ||
      (rc = check_heads(what, "out", out)) || (rest != nullptr && (rc = check_heads(what, "rest", rest))) ||
      (rc = check_heads(what, "grad_out", grad_out)) ||
      (rc = check_heads(what, "dq", dq)) || (rc = check_heads(what, "dk", dk)) || (rc = check_heads(what, "dv", dv)))
    return rc;
  PKM_REQUIRE(lse != nullptr, PKM_ERR_INVALID_ARGUMENT, "%s: lse is NULL", what);
  plan_far(&a);
  PKM_REQUIRE(workspace != nullptr && workspace_bytes >= (size_t)(delta_bytes(a) + far_bytes(a)), PKM_ERR_WORKSPACE,
              "%s: workspace too small", what);
  PKM_REQUIRE(((uintptr_t)workspace & 15) == 0, PKM_ERR_INVALID_ARGUMENT, "%s: workspace is not 16-byte aligned", what);
  a.q = heads(q), a.k = heads(k), a.v = heads(v), a.o = heads(out), a.dO = heads(grad_out);
  a.dq = heads(dq), a.dk = heads(dk), a.dv = heads(dv);
  if (rest != nullptr) a.rest = heads(rest);
  a.starts = starts, a.ends = ends, a.lse = const_cast<float*>(lse), a.delta = (float*)workspace;
  a.far = (float*)((uint8_t*)workspace + delta_bytes(a));
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKM_DTYPE_BF16) {
    dim == 128 ? launch_bwd<bf16_t, 128>(a, st) : launch_bwd<bf16_t, 64>(a, st);
  } else {
    dim == 128 ? launch_bwd<f16_t, 128>(a, st) : launch_bwd<f16_t, 64>(a, st);
  }
  return pkm_check_launch(what);
}
