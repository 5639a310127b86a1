// Causal attention through a sliding window, with a few first tokens that stay
// visible (sinks), over padded batches: forward and backward.
//
// Key j is visible to the query at position p of a sequence of tokens
// [start, end) if start <= j <= p < end and (p - j < window or j - start < sinks).
//   o_p = sum_j P_pj v_j,  P_pj = exp(scale q_p.k_j - lse_p),  lse_p = log sum_j exp(scale q_p.k_j)
//   dV = P^T dO,  dS = P (dO V^T - delta),  delta_p = dO_p.o_p,  dQ = scale dS K,  dK = scale dS^T Q
// Positions inside the kernels are relative to the sequence's start.
#include "attn_common.h"

namespace pkm {
namespace {

constexpr int kThreads = 256;  // 4 waves
constexpr int kTile = 64;      // rows of an LDS tile

struct AttnArgs {
  Heads q, k, v, o, dO, dq, dk, dv;
  float* lse;    // [batch, q_heads, tokens], in units of log2; +inf where nothing is visible
  float* delta;  // [batch, q_heads, tokens]
  const int* starts;
  const int* ends;
  int batch, q_heads, kv_heads, tokens;
  int window, sinks;  // window in [1, tokens] (tokens: no window), sinks in [0, tokens]
  int pack;           // query heads of one key head that share a workgroup: 1, 2 or 4
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
// lane holds one query's weights; O^T = V^T P^T takes them as they lie.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void window_fwd_kernel(const AttnArgs a) {
  constexpr int KS = D / 16, DT = D / 32, TB = kTile * D * 2;
  __shared__ __align__(16) uint8_t smem[2 * 2 * TB];
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
    const lds_u8* ktile = lds + (it & 1) * 2 * TB;
    const lds_u8* vtile = ktile + TB;
    if (it + 1 < tiles.count) {
      const int t1 = tiles.tile(it + 1) * kTile;
      lds_u8* next = lds + ((it + 1) & 1) * 2 * TB;
      tl.load(next, kbase + (int64_t)t1 * kstride, kstride, seq.n - t1, tid);
      tl.load(next + TB, vbase + (int64_t)t1 * vstride, vstride, seq.n - t1, tid);
    }
    if (p0 <= p1 && any_visible(p0, p1, j0, j0 + kTile - 1, W, S)) {
      f32x16_t s[2] = {};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < KS; ++i) s[kb] = mfma32<T>(frag_rows<D>(ktile, 32 * kb, i, lane), q[i], s[kb]);
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
      const float mc = (top == -INFINITY ? 0.f : top) * c;
      if (__any(top > m)) {
        const float f = exp2_raw(__builtin_fmaf(m, c, -mc));
        sum *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[t][i] *= f;
        m = top;
      }
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
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = mfma32<T>(frag_cols<D>(vtile, 16 * i, t, lane), pf[i], o[t]);
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
  store_row<T, D>(a.o.at(qb.b, qb.head, row), o, some ? 1.f / sum : 0.f, lane);
  if (a.lse && h == 0) {
    a.lse[((int64_t)qb.b * a.q_heads + qb.head) * a.tokens + row] =
        some ? m * c + __builtin_amdgcn_logf(sum) : INFINITY;
  }
}

// ---------------------------------------------------------------------------
// Backward, dQ: as the forward, dS^T = P^T (V dO^T - delta), dQ^T = K^T dS^T.
//
// delta comes from the rounded output. What that puts into a row's dS adds up to
// sum_j dS_j (which is 0), so the sum corrects the delta that dK reads. dS enters its
// product as two 16-bit numbers, itself rounded and the rest: keys have a common part,
// which the exact dS, whose sum is 0, cancels and the roundings of one would not (relative error
// of dQ 2.7e-3 with one, 2.0e-3 with two in bf16, where the result's own rounding is 1.7e-3).
// ---------------------------------------------------------------------------
template <typename T, int D>
__device__ void window_dq_block(const AttnArgs& a, int id, uint8_t* smem) {
  constexpr int KS = D / 16, DT = D / 32, TB = kTile * D * 2;
  lds_u8* const lds = (lds_u8*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = lane & 31, h = lane >> 5;
  const QueryBlock qb(a, id, wave);
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
  const float lse = live ? a.lse[at] : INFINITY;
  float delta = 0.f, sum = 0.f;
  const uint8_t* orow = live ? a.o.at(qb.b, qb.head, row) : nullptr;
#pragma unroll
  for (int s = 0; s < KS; ++s)
    delta = vec_dot<T>(__builtin_bit_cast(uint4, frag_global<D>(orow, s, lane)), __builtin_bit_cast(uint4, g[s]), delta);
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
    const lds_u8* ktile = lds + (it & 1) * 2 * TB;
    const lds_u8* vtile = ktile + TB;
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
#pragma unroll
        for (int i = 0; i < KS; ++i) s = mfma32<T>(frag_rows<D>(ktile, 32 * kb, i, lane), q[i], s);
#pragma unroll
        for (int i = 0; i < KS; ++i) dp = mfma32<T>(frag_rows<D>(vtile, 32 * kb, i, lane), g[i], dp);
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
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          frag_t f, r;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[8 * i + 2 * e], y = s[8 * i + 2 * e + 1];
            f[e] = pack2<T>(x, y);
            r[e] = pack2<T>(x - unpack1<T>(f[e] & 0xffffu), y - unpack1<T>(f[e] >> 16));
          }
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            const frag_t kt = frag_cols<D>(ktile, 32 * kb + 16 * i, t, lane);
            dq[t] = mfma32<T>(kt, f, dq[t]);
            dq[t] = mfma32<T>(kt, r, dq[t]);
          }
        }
      }
    }
    tile_wait();
    __syncthreads();
  }
  sum += swap_halves(sum);
  if (row >= a.tokens) return;
  if (live && h == 0) a.delta[at] = delta + sum;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[t][i] = live ? dq[t][i] : 0.f;
  store_row<T, D>(a.dq.at(qb.b, qb.head, row), dq, a.scale, lane);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void window_dq_kernel(const AttnArgs a) {
  __shared__ __align__(16) uint8_t smem[2 * 2 * kTile * D * 2];
  window_dq_block<T, D>(a, blockIdx.x, smem);
}

// ---------------------------------------------------------------------------
// Backward, dK and dV: 4 waves of 32 keys each; the tiles hold 64 queries and
// their dO, of every query head of the key head in turn (a shared head's
// gradient is summed in registers, in a fixed order).
// ---------------------------------------------------------------------------
template <typename T, int D>
__device__ void window_dkv_block(const AttnArgs& a, int id, uint8_t* smem) {
  constexpr int KS = D / 16, DT = D / 32, TB = kTile * D * 2, BUF = 2 * TB + 2 * kTile * 4;
  lds_u8* const lds = (lds_u8*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = lane & 31, h = lane >> 5;
  const int pairs = a.batch * a.kv_heads, pair = id % pairs;
  const int b = pair / a.kv_heads, kv = pair % a.kv_heads, G = a.q_heads / a.kv_heads;
  const int first = id / pairs * 128;  // the key block's rows; the first ones are read by most queries
  const Span seq = sequence(a, b);
  const int W = a.window, S = a.sinks, n = seq.n;
  const int row = first + 32 * wave + l;
  const int key = row - seq.start;
  const bool live = row < a.tokens && key >= 0 && key < n;
  const int k0 = max(first + 32 * wave - seq.start, 0), k1 = min(first + 32 * wave + 31 - seq.start, n - 1);
  // the queries that see the block: from its first key to the window's end of its last, or all of them
  const int b0 = max(first - seq.start, 0), b1 = min(first + 127 - seq.start, n - 1);
  int tile0 = 0, count = 0;
  if (b0 <= b1) {
    const int last = b0 < S ? n - 1 : min(n - 1, b1 + W - 1);
    tile0 = b0 / kTile;
    count = last / kTile + 1 - tile0;
  }
  const int total = count * G;

  frag_t k[KS], v[KS];
  const uint8_t* krow = live ? a.k.at(b, kv, row) : nullptr;
  const uint8_t* vrow = live ? a.v.at(b, kv, row) : nullptr;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    k[s] = frag_global<D>(krow, s, lane);
    v[s] = frag_global<D>(vrow, s, lane);
  }
  const TileLoad<D, kTile> tl(tid);
  const uint32_t qstride = (uint32_t)(2 * a.q.token), gstride = (uint32_t)(2 * a.dO.token);
  float aux = 0.f;  // threads 0 .. 63 carry a tile's lse, 64 .. 127 its delta
  const auto load = [&](int i) {
    const int head = kv * G + i / count, t0 = (tile0 + i % count) * kTile;
    lds_u8* buf = lds + (i & 1) * BUF;
    tl.load(buf, a.q.at(b, head, seq.start + t0), qstride, n - t0, tid);
    tl.load(buf + TB, a.dO.at(b, head, seq.start + t0), gstride, n - t0, tid);
    if (tid < 2 * kTile) {
      const int r = tid & (kTile - 1);
      const float* from = tid < kTile ? a.lse : a.delta;
      aux = t0 + r < n ? from[((int64_t)b * a.q_heads + head) * a.tokens + seq.start + t0 + r]
                       : (tid < kTile ? INFINITY : 0.f);
    }
  };
  const auto store = [&](int i) {
    lds_u8* buf = lds + (i & 1) * BUF;
    if (tid < 2 * kTile) *(__attribute__((address_space(3))) float*)(buf + 2 * TB + 4 * tid) = aux;
  };

  f32x16_t dk[DT] = {}, dv[DT] = {};
  const float c = a.scale * 1.44269504f;
  if (total > 0) {
    load(0);
    store(0);
  }
  tile_wait();
  __syncthreads();
  for (int it = 0; it < total; ++it) {
    const int p0 = (tile0 + it % count) * kTile;
    const lds_u8* qtile = lds + (it & 1) * BUF;
    const lds_u8* gtile = qtile + TB;
    const lds_u8* stats = gtile + TB;
    if (it + 1 < total) load(it + 1);
    if (k0 <= k1) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const int pa = p0 + 32 * qb;
        if (!any_visible(pa, pa + 31, k0, k1, W, S)) continue;
        f32x16_t s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < KS; ++i) s = mfma32<T>(frag_rows<D>(qtile, 32 * qb, i, lane), k[i], s);
#pragma unroll
        for (int i = 0; i < KS; ++i) dp = mfma32<T>(frag_rows<D>(gtile, 32 * qb, i, lane), v[i], dp);
        if (!all_visible(pa, pa + 31, k0, k1, W, S)) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[i] = visible(pa + 8 * (i >> 2) + 4 * h + (i & 3), key, W, S) ? s[i] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4_t lse = *(const lds_f32x4*)(stats + 4 * (32 * qb + 8 * e + 4 * h));
          const f32x4_t delta = *(const lds_f32x4*)(stats + 4 * (kTile + 32 * qb + 8 * e + 4 * h));
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 4 * e + r;
            s[i] = exp2_raw(__builtin_fmaf(s[i], c, -lse[r]));
            dp[i] = s[i] * (dp[i] - delta[r]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          frag_t pf, sf;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pf[e] = pack2<T>(s[8 * i + 2 * e], s[8 * i + 2 * e + 1]);
            sf[e] = pack2<T>(dp[8 * i + 2 * e], dp[8 * i + 2 * e + 1]);
          }
#pragma unroll
          for (int t = 0; t < DT; ++t) dv[t] = mfma32<T>(frag_cols<D>(gtile, 32 * qb + 16 * i, t, lane), pf, dv[t]);
#pragma unroll
          for (int t = 0; t < DT; ++t) dk[t] = mfma32<T>(frag_cols<D>(qtile, 32 * qb + 16 * i, t, lane), sf, dk[t]);
        }
      }
    }
    if (it + 1 < total) store(it + 1);
    tile_wait();
    __syncthreads();
  }
  if (row >= a.tokens) return;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dk[t][i] = live ? dk[t][i] : 0.f;
      dv[t][i] = live ? dv[t][i] : 0.f;
    }
  store_row<T, D>(a.dk.at(b, kv, row), dk, a.scale, lane);
  store_row<T, D>(a.dv.at(b, kv, row), dv, 1.f, lane);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, 1) void window_dkv_kernel(const AttnArgs a) {
  __shared__ __align__(16) uint8_t smem[2 * (2 * kTile * D * 2 + 2 * kTile * 4)];
  window_dkv_block<T, D>(a, blockIdx.x, smem);
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
  PKM_REQUIRE(tokens < (1 << 24) && batch * q_heads < (1 << 24) && batch * q_heads * ((tokens + 31) / 32) < (1ll << 31),
              PKM_ERR_UNSUPPORTED, "%s: too many tokens or heads", what);
  a->batch = (int)batch;
  a->q_heads = (int)q_heads;
  a->kv_heads = (int)kv_heads;
  a->tokens = (int)tokens;
  a->window = (int)(window == 0 || window > tokens ? tokens : window);
  a->sinks = (int)(sinks > tokens ? tokens : sinks);
  a->scale = scale;
  const int64_t share = q_heads / kv_heads;
  a->pack = share % 4 == 0 ? 4 : share % 2 == 0 ? 2 : 1;
  return PKM_OK;
}

unsigned query_blocks(const AttnArgs& a) {
  const int rows = 128 / a.pack;
  return (unsigned)(a.batch * (a.q_heads / a.pack) * ((a.tokens + rows - 1) / rows));
}

template <typename T, int D>
void launch_fwd(const AttnArgs& a, hipStream_t st) {
  window_fwd_kernel<T, D><<<query_blocks(a), kThreads, 0, st>>>(a);
}

template <typename T, int D>
void launch_bwd(const AttnArgs& a, hipStream_t st) {
  window_dq_kernel<T, D><<<query_blocks(a), kThreads, 0, st>>>(a);  // and delta
  window_dkv_kernel<T, D><<<(unsigned)(a.batch * a.kv_heads * ((a.tokens + 127) / 128)), kThreads, 0, st>>>(a);
}

}  // namespace
}  // namespace pkm

using namespace pkm;

extern "C" int pkm_window_attn_fwd(const pkm_heads_t* q, const pkm_heads_t* k, const pkm_heads_t* v,
                                   const int32_t* starts, const int32_t* ends, int64_t batch, int64_t q_heads,
                                   int64_t kv_heads, int64_t tokens, int64_t dim, int dtype, int64_t window,
                                   int64_t sinks, float scale, const pkm_heads_t* out, float* lse, void* stream) {
  const char* what = "pkm_window_attn_fwd";
  AttnArgs a = {};
  int rc = fill_args(what, &a, batch, q_heads, kv_heads, tokens, dim, dtype, window, sinks, scale);
  if (rc != PKM_OK) return rc;
  if (batch == 0 || tokens == 0) return PKM_OK;
  if ((rc = check_heads(what, "q", q)) || (rc = check_heads(what, "k", k)) || (rc = check_heads(what, "v", v)) ||
      (rc = check_heads(what, "out", out)))
    return rc;
  a.q = heads(q), a.k = heads(k), a.v = heads(v), a.o = heads(out);
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
  (void)kv_heads, (void)dim, (void)window, (void)sinks;
  return batch <= 0 || q_heads <= 0 || tokens <= 0 ? 0 : (size_t)(batch * q_heads * tokens) * sizeof(float);
}

extern "C" int pkm_window_attn_bwd(const pkm_heads_t* q, const pkm_heads_t* k, const pkm_heads_t* v,
                                   const pkm_heads_t* out, const float* lse, const pkm_heads_t* grad_out,
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
      (rc = check_heads(what, "out", out)) || (rc = check_heads(what, "grad_out", grad_out)) ||
      (rc = check_heads(what, "dq", dq)) || (rc = check_heads(what, "dk", dk)) || (rc = check_heads(what, "dv", dv)))
    return rc;
  PKM_REQUIRE(lse != nullptr, PKM_ERR_INVALID_ARGUMENT, "%s: lse is NULL", what);
  PKM_REQUIRE(workspace != nullptr && workspace_bytes >= pkm_window_attn_bwd_workspace_size(batch, q_heads, kv_heads, tokens, dim, window, sinks),
              PKM_ERR_WORKSPACE, "%s: workspace too small", what);
  a.q = heads(q), a.k = heads(k), a.v = heads(v), a.o = heads(out), a.dO = heads(grad_out);
  a.dq = heads(dq), a.dk = heads(dk), a.dv = heads(dv);
  a.starts = starts, a.ends = ends, a.lse = const_cast<float*>(lse), a.delta = (float*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKM_DTYPE_BF16) {
    dim == 128 ? launch_bwd<bf16_t, 128>(a, st) : launch_bwd<bf16_t, 64>(a, st);
  } else {
    dim == 128 ? launch_bwd<f16_t, 128>(a, st) : launch_bwd<f16_t, 64>(a, st);
  }
  return pkm_check_launch(what);
}
