// Softmax cross entropy of a linear layer over a large vocabulary, forward and backward, without the logits in memory,
// gfx950.
//
//   l_jv = <x_j, W_v>    lse_j = log sum_v exp l_jv    loss_j = lse_j - l_j,y_j
//   d_jv = g_j (exp(l_jv - lse_j) - [v = y_j])    dx_j = sum_v d_jv W_v    dW_v = sum_j d_jv x_j
//
// for the tokens whose label lies in [0, vocab) and is not the ignored one: these are copied side by side first ("kept"
// tokens, padded to whole 128-byte lines), so that nothing is computed for the others and what they hold (NaN) reaches
// nothing. The number of kept tokens stays on the device.
//
// Forward: one product, [vocab, tokens], whose epilogue sums the exponentials of a tile and drops the logits. Backward: for a
// piece of the vocabulary after the other the same product again, whose epilogue leaves d in 16 bits, and from it the
// piece's rows of dW, whole, and its part of dx, added up in float32. That is 8 n V D operations where keeping the logits
// would take 6. What bounds all of it are the matrix cores.
//
// The three products are one kernel (ce_product): tiles of 256 x 256 results by 8 waves (2 x 4, each 128 x 64 in 32x32x16
// products), 64 deep, in two stages of 64 KB of LDS that buffer loads fill without registers. A wave reads the operands of
// a step of 16 while the matrix cores work on the one before, across tiles and also across results: the grid is one
// workgroup a CU, and the next result's tiles load while this one's epilogue runs. One barrier a 64.
//
// Measured, 16384 tokens, 151936 entries, 1024 wide, bf16: the forward's product 4.16 to 4.48 ms (several cards; 1140 to 1225
// TFLOP/s), of a piece of 15360 entries d 0.49, dW 0.44 and dx 0.42 ms (1040 to 1200); beside them 0.1 ms (count and copy of the
// tokens 23 us, join of the tiles' sums 47, dx's rounding 50). The matrix cores are busy 52 to 61 % of the cycles at 1.6 to 2.0 GHz;
// plain library products of the pieces' shapes take 0.457, 0.668 and 0.444 ms at 1.5 to 1.64 GHz and 50 to 70 %: the clock
// falls as the load rises, and neither fewer LDS cycles (bank conflicts were half of them) nor loads spread between the
// products moved the time.
//
// d lies as the epilogue's registers hold it, in blocks of 16 vocabulary entries x 32 tokens (1 KB, 16 bytes a lane): dx's
// product reads a block as a matrix operand as it is, dW's through the transposing LDS reads.
#include "attn_common.h"

namespace pkm {
namespace {

constexpr int kTile = 256, kDepth = 64, kHalf = 32768, kStage = 2 * kHalf;
constexpr int kThreads = 512;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

enum Product { kLoss, kGrads, kDx, kDw };

// What a result of dx's or dW's product is multiplied by.
struct Scale {
  const float* value;  // ce_weights'
  const float* grad;   // or the gradient of the sum or the mean
  const int32_t* count;
  float lift;
  int32_t mean;
  __device__ __forceinline__ float operator()() const {
    return grad ? *grad / ((mean ? (float)max(*count, 1) : 1.f) * lift) : *value;
  }
};

struct CeArgs {
  const uint8_t* x;  // kept tokens [npad, dpad]
  const uint8_t* w;
  uint8_t* d;  // blocks of a piece [piece / 16][npad / 32][1 KB]
  int64_t x_stride, w_stride;  // bytes
  const int32_t* count;  // kept tokens
  const int32_t* label;  // [npad]
  const float* ref;      // [npad] the label's logit to a few roundings, the softmax sums' reference
  float* target;         // [npad] the label's logit as the product gives it
  const float* loss;     // [npad]
  const float* lse;      // [npad]
  const float* weight;   // [npad] of the tokens' gradients, or NULL: `lift` for all
  const float* unit;     // [npad] what a token's row of dx is multiplied by, or NULL: `scale` for all
  float2* sums;          // [2 * vocab tiles][npad] reference and sum of exponentials
  float* parts;          // [splits][whole tiles' rows][dcols] float32: of dx, or of dW where its sum is split
  uint8_t* dw;           // [vocab][dim]
  Scale scale;
  int64_t vocab, v0;  // v0: the piece's first entry
  int32_t piece, dim, npad, dcols, splits, add;
  int32_t pair;  // few tokens: d as two numbers of 16 bits, the second ones in the token slots behind the first
};

__device__ __forceinline__ int perm16(int k) { return ((k & 3) << 2) | ((k >> 2) & 3); }

// 64 lanes' 16 bytes each from base + their offset to LDS at `to` and on, side by side; vmcnt counts them, the compiler does not.
// The descriptor may come from a vector instruction (a lane read, a spilled scalar), which a memory instruction has to
// follow by 5 states: inside the asm only we see to that.
__device__ __forceinline__ void load16(const uint8_t* base, lds_u8* to, uint32_t offset) {
  const u32x4_t rs = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)base),
                      (uint32_t)__builtin_amdgcn_readfirstlane((int)((uintptr_t)base >> 32)), 0x7fffffffu, 0x00020000u};
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"((uint32_t)(uintptr_t)to), "v"(offset), "s"(rs)
               : "memory");
}

// The operands' tiles: how a wave loads its four KB of one and reads a matrix operand from it.
// L = wave + 8 n is the KB that load n fills.

// [256 rows][64 numbers] of a matrix whose rows hold the summed index: 128 bytes a row, chunks permuted by row / 2, so that
// 16 rows' chunks fall on all 64 banks. Rows
// behind the last repeat it; chunks behind the row's end repeat the last one, against zeros of the other operand.
struct RowsTile {
  const uint8_t* base;
  uint32_t off[4];
  int chunk;
  __device__ __forceinline__ void at(const uint8_t* p, int64_t stride, int64_t row0, int64_t rows, int wave, int lane) {
    base = p + row0 * stride;
    const int64_t last = rows - 1 - row0;
    chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
#pragma unroll
    for (int n = 0; n < 4; ++n) off[n] = (uint32_t)(min((int64_t)(8 * wave + 64 * n + (lane >> 3)), last) * stride);
  }
  __device__ __forceinline__ void load(lds_u8* to, int n, int step, int chunks, int wave) const {
    const uint32_t c = (uint32_t)min(step * 8 + chunk, chunks - 1) << 4;
    load16(base, to + (wave + 8 * n) * 1024, off[n] + c);
  }
};
__device__ __forceinline__ uint32_t rows_lane(int lane) {
  return (lane & 31) * 128 + (((lane >> 5) ^ ((lane >> 1) & 7)) << 4);
}
__device__ __forceinline__ frag_t rows_frag(uint32_t at, int t, int s) {
  return *(const lds_u32x4*)(uintptr_t)((at ^ (uint32_t)(s << 5)) + t * 4096);
}

// [64 rows][256 columns] of a matrix whose rows are the summed index: 512 bytes a row, chunks permuted by the row.
struct ColsTile {
  const uint8_t* base;
  uint32_t col;
  __device__ __forceinline__ void at(const uint8_t* p, int col0, int chunks, int wave, int lane) {
    base = p;
    col = (uint32_t)min(col0 / 8 + ((lane & 31) ^ perm16(2 * wave + (lane >> 5))), chunks - 1) << 4;
  }
  __device__ __forceinline__ void load(lds_u8* to, int n, int step, int64_t stride, int64_t rows, int wave, int lane) const {
    const uint8_t* const b = base + (int64_t)step * kDepth * stride;
    const int last = (int)min(rows - 1 - (int64_t)step * kDepth, (int64_t)kDepth);
    load16(b, to + (wave + 8 * n) * 1024, (uint32_t)min(2 * wave + 16 * n + (lane >> 5), last) * (uint32_t)stride + col);
  }
};
__device__ __forceinline__ uint32_t cols_lane(int lane) {
  const int l = lane & 15, h = lane >> 5, g = (lane >> 4) & 1;
  return (4 * h + (l >> 2)) * 512 + (((2 * g + ((l & 3) >> 1)) ^ (((l >> 2) << 2) | h)) << 4) + (l & 1) * 8;
}
__device__ __forceinline__ frag_t two_tr(uint32_t p, uint32_t q) {
  const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)p);
  const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)q);
  const u32x2_t x = __builtin_bit_cast(u32x2_t, a), y = __builtin_bit_cast(u32x2_t, b);
  return (frag_t){x[0], x[1], y[0], y[1]};
}
// Summed index in the order 4 h + 0..3, 8 + 4 h + 0..3, which is how d's blocks have it.
__device__ __forceinline__ frag_t cols_frag(uint32_t at, int t, int s) {
  return two_tr((at ^ (uint32_t)(t << 6)) + s * 8192, (at ^ (uint32_t)((t << 6) | 32)) + s * 8192 + 4096);
}

// Where a block of d, of entries 16 g .. 16 g + 15, holds lane (h, token)'s 16 bytes: the halves 64 bytes apart in a
// 128-byte line and neighbouring blocks 128 bytes in 256, so that a transposing read falls on all 64 banks.
__device__ __forceinline__ constexpr int block_lane(int g, int h, int t) { return 32 * h + (t ^ (h << 2) ^ ((g & 1) << 3)); }

// d as dx's operand: 256 tokens, 64 vocabulary entries. Block (entries n, tokens wave).
__device__ __forceinline__ void load_tokens(const uint8_t* d, lds_u8* to, int n, int step, int tile, int npad, int wave,
                                            int lane) {
  const uint32_t row = (uint32_t)(npad / 32) * 1024;
  const uint8_t* const b = d + ((int64_t)step * 4 + n) * row + (int64_t)tile * 8192 + wave * 1024;
  load16(b, to + (wave + 8 * n) * 1024, lane * 16);
}
__device__ __forceinline__ uint32_t tokens_lane(int lane) { return block_lane(0, lane >> 5, lane & 31) * 16; }
__device__ __forceinline__ frag_t tokens_frag(uint32_t at, int t, int s) {
  return *(const lds_u32x4*)(uintptr_t)((at ^ (uint32_t)((s & 1) << 7)) + s * 8192 + t * 1024);
}

// d as dW's operand: 256 vocabulary entries, 64 tokens. Block (entries L / 2, tokens L % 2).
__device__ __forceinline__ void load_entries(const uint8_t* d, lds_u8* to, int n, int step, int tile, int npad, int wave,
                                             int lane) {
  const int L = wave + 8 * n;
  const uint32_t row = (uint32_t)(npad / 32) * 1024;
  const uint8_t* const b = d + ((int64_t)tile * 16 + (L >> 1)) * row + (int64_t)step * 2048 + (L & 1) * 1024;
  load16(b, to + L * 1024, lane * 16);
}
__device__ __forceinline__ uint32_t entries_lane(int lane) {
  const int l = lane & 15, h = lane >> 5, g = (lane >> 4) & 1, p = l & 3;
  return g * 2048 + block_lane(g, p & 1, 4 * h + (l >> 2)) * 16 + 8 * (p >> 1);
}
__device__ __forceinline__ frag_t entries_frag(uint32_t at, int t, int s) {
  const int to = t * 4096 + (s >> 1) * 1024 + (s & 1) * 256;
  return two_tr(at + to, (at ^ 128) + to);
}

// Results of a product go in blocks of 2^lg_m x 2^lg_n tiles, 32 at most, to workgroups of one XCD, so that these share the
// tiles' rows in its L2; blocks run along N first.
struct Blocks {
  int lg_m = 0, lg_n, m, n;  // m, n: how many
  __host__ __device__ Blocks(int64_t tiles_m, int64_t tiles_n) {
    lg_n = tiles_n >= 4 ? 2 : tiles_n >= 2 ? 1 : 0;
    while (lg_m < 5 - lg_n && (1 << lg_m) < tiles_m) ++lg_m;
    m = (int)((tiles_m + (1 << lg_m) - 1) >> lg_m);
    n = (int)((tiles_n + (1 << lg_n) - 1) >> lg_n);
  }
  __host__ __device__ int64_t results() const { return ((int64_t)m * n) << (lg_m + lg_n); }
};

// Splits of a product's sum over `steps`, so that few results fill the CUs once: 8 steps at least each, which outweigh the
// partial results' way through memory.
__host__ __device__ inline int splits_of(int64_t tiles_m, int64_t tiles_n, int64_t steps) {
  const int64_t results = Blocks(tiles_m, tiles_n).results();
  int64_t n = results < 1 ? 1 : 256 / results;
  if (n > steps / 8) n = steps / 8;
  return n < 1 ? 1 : (int)n;
}

struct Order {
  Blocks blocks;
  int m, n, k, splits, total, share;
  __device__ __forceinline__ Order(int m_, int n_, int k_, int splits_) : blocks(m_, n_), m(m_), n(n_), k(k_), splits(splits_) {
    total = (int)blocks.results() * splits;
    share = min(32, (total + 7) / 8);  // results of an XCD at a time
  }
};
struct Result {
  int i, m, n, split, k0, k1;  // i: the order's place; steps [k0, k1)
  __device__ __forceinline__ bool next(const Order& o, bool first) {
    const int b = blockIdx.x, xcd = b & 7, own = b >> 3;
    if (first) {
      if (own >= o.share) return false;
      i = xcd * o.share + own;
    } else {
      i += 8 * o.share;
    }
    for (; i < o.total; i += 8 * o.share) {
      const int lg_m = o.blocks.lg_m, lg = lg_m + o.blocks.lg_n;
      const int within = i & ((1 << lg) - 1), block = i >> lg, rest = block / o.splits;
      split = block - rest * o.splits;
      m = ((rest / o.blocks.n) << lg_m) + (within & ((1 << lg_m) - 1));
      n = ((rest % o.blocks.n) << o.blocks.lg_n) + (within >> lg_m);
      if (m >= o.m || n >= o.n) continue;
      k0 = (int)((int64_t)o.k * split / o.splits);
      k1 = (int)((int64_t)o.k * (split + 1) / o.splits);
      if (k1 > k0) return true;
    }
    return false;
  }
};

// The epilogues. A wave's 128 x 64: acc[t][u][i] is row 32 t + 8 (i / 4) + 4 h + i % 4, column 32 u + lane % 32.
typedef f32x16_t acc_t[4][2];

__device__ __forceinline__ constexpr int row_of(int t, int i) { return 32 * t + 8 * (i >> 2) + (i & 3); }  // but 4 h

// Nothing moves across: a batch of registers is done with before the next begins.
__device__ __forceinline__ void batch() { __builtin_amdgcn_sched_barrier(0); }

// Results behind the vocabulary's end, `left` rows from the wave's first: -infinity in their place.
template <int MT, int NU>
__device__ __forceinline__ void cut(f32x16_t (&acc)[MT][NU], int64_t left, int h) {
  if (left >= 32 * MT) return;
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    int most = (int)left - 4 * h;
    asm volatile("" : "+v"(most));  // compared anew for each half: 64 masks would not fit the scalar registers
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][u][i] = row_of(t, i) < most ? acc[t][u][i] : -INFINITY;
  }
}

// 0 for the label's row, else 1.
__device__ __forceinline__ float others(int row, float yr) { return fminf((row - yr) * (row - yr), 1.f); }

// The sum of the exponentials of a wave's entries for the lane's token of column block u, against the token's reference: the
// label's logit, whose own exponential is 1, so that what underflows beside it is nothing. Where a sum reaches 2^96, the
// entries' own largest logit takes the reference's place: up to 2^25 sums of 32 entries or more (fewer than 2^30 in all) are
// added up against one reference later (joined), and stay below 2^121. The reference's product with log2(e) is rounded once for
// all entries; what that adds to all exponents alike comes off the sum.
// OWN: the label may be among the entries, yr rows (less 4 h) below the wave's first: its logit goes to `target`, its exponential
// is left out. A loss near 0 is the logarithm of 1 + the others' exponentials, which a 1 among them would round. Left out by a
// factor 0 or 1 (others): the masks of 64 comparisons would not fit the scalar registers.
template <bool OWN, int MT, int NU>
__device__ __forceinline__ float2 sum_over(const f32x16_t (&acc)[MT][NU], int u, float ref, int yr, float* target) {
  float sum = 0.f, z = -INFINITY;
  const float c = -ref * kLog2e, y = (float)yr;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = exp2_raw(__builtin_fmaf(acc[t][u][i], kLog2e, c));
      if constexpr (OWN) {
        const float w = others(row_of(t, i), y);
        z = fmaxf(z, __builtin_fmaf(w, -3e38f, acc[t][u][i]));
        sum = __builtin_fmaf(e, w, sum);
      } else {
        sum += e;
      }
    }
    batch();
  }
  if constexpr (OWN) {
    if (yr >= 0 && yr < 32 * MT && (yr & 4) == 0) *target = z < -2e38f ? -INFINITY : z;  // an infinite one, beside the others
  }
  sum += swap_halves(sum);
  sum -= sum * (__builtin_fmaf(ref, kLog2e, c) * kLn2);
  const bool over = !(sum < 0x1p96f);
  if (__any(over)) {
    float top = -3e38f;  // finite, for entries that are all -infinity
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, acc[t][u][i]);
    top = fmaxf(top, swap_halves(top));
    float own = 0.f;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = exp2_raw((acc[t][u][i] - top) * kLog2e);
        own = OWN ? __builtin_fmaf(e, others(row_of(t, i), y), own) : own + e;
      }
      batch();
    }
    own += swap_halves(own);
    if (over) ref = top, sum = own;
  }
  return make_float2(ref, sum);
}
template <int MT, int NU>
__device__ __forceinline__ float2 sum_of(const f32x16_t (&acc)[MT][NU], int u, float ref, int yr, float* target) {
  if (__any(yr >= 0 && yr < 32 * MT)) return sum_over<true>(acc, u, ref, yr, target);
  return sum_over<false>(acc, u, ref, yr, target);
}

// Two such sums as one.
__device__ __forceinline__ float2 joined(float2 a, float2 b) {
  if (b.x > a.x) return make_float2(b.x, a.y * exp2_raw((a.x - b.x) * kLog2e) + b.y);
  return make_float2(a.x, a.y + (b.x == a.x ? b.y : b.y * exp2_raw((b.x - a.x) * kLog2e)));
}

__device__ __forceinline__ void end_loss(const CeArgs& a, acc_t& acc, const Result& r, int wave, int lane) {
  const int h = lane >> 5, v0 = r.m * kTile + (wave >> 2) * 128;
  cut(acc, a.vocab - v0, h);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = r.n * kTile + (wave & 3) * 64 + 32 * u + (lane & 31);
    const float2 sum = sum_of(acc, u, a.ref[j], a.label[j] - v0 - 4 * h, a.target + j);
    if (h == 0) a.sums[(int64_t)(2 * r.m + (wave >> 2)) * a.npad + j] = sum;
  }
}

// The label's d: exp(l - lse) - 1 = exp(- loss) - 1, with its weight.
__device__ __forceinline__ float label_d(float loss, float weight) { return expm1f(-loss) * weight; }

// Two numbers of 16 bits for each of f: its rounding and, `low`, the rounding of what that left.
template <typename T>
__device__ __forceinline__ u32x4_t rounded(const float (&f)[8], bool low) {
  u32x4_t x;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = pack2<T>(f[2 * e], f[2 * e + 1]);
    if (low) x[e] = pack2<T>(f[2 * e] - unpack1<T>(x[e] & 0xffffu), f[2 * e + 1] - unpack1<T>(x[e] >> 16));
  }
  return x;
}

// d of a wave's entries, from v0 of the piece on, for the lane's token j of column block u, rounded, in blocks; with `second`,
// what the rounding left in the blocks that many bytes further.
// c: - lse log2(e), -infinity for a token that is not kept; y: the label's place from v0 on.
template <typename T, int MT, int NU>
__device__ __forceinline__ void grads_of(const CeArgs& a, const f32x16_t (&acc)[MT][NU], int u, int64_t v0, int j, float c,
                                         float weight, int64_t y, float loss, int64_t second, int lane) {
  const int h = lane >> 5;
  const int64_t row = (int64_t)(a.npad / 32) * 1024;
  uint8_t* const to = a.d + (v0 / 16) * row + (int64_t)(j >> 5) * 1024;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = exp2_raw(__builtin_fmaf(acc[t][u][8 * s + e], kLog2e, c)) * weight;
      uint8_t* const at = to + (2 * t + s) * row + block_lane(s, h, lane & 31) * 16;
      *(u32x4_t*)at = rounded<T>(f, false);
      if (second) *(u32x4_t*)(at + second) = rounded<T>(f, true);
    }
    batch();
  }
  // the label's number takes the place of the one written above
  const bool own = y >= 0 && y < 32 * MT;
  if (__any(own)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (own && h == 0) {
      const float x = label_d(loss, weight);
      uint8_t* const at =
          to + (y >> 4) * row + block_lane((y >> 4) & 1, (y >> 2) & 1, lane) * 16 + ((y >> 3) & 1) * 8 + (y & 3) * 2;
      const uint32_t high = pack2<T>(x, x) & 0xffffu;
      *(uint16_t*)at = (uint16_t)high;
      if (second) *(uint16_t*)(at + second) = (uint16_t)pack2<T>(x - unpack1<T>(high), 0.f);
    }
  }
}

template <typename T>
__device__ __forceinline__ void end_grads(const CeArgs& a, acc_t& acc, const Result& r, int count, int wave, int lane) {
  const int64_t v0 = r.m * kTile + (wave >> 2) * 128;
  cut(acc, a.vocab - a.v0 - v0, lane >> 5);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = r.n * kTile + (wave & 3) * 64 + 32 * u + (lane & 31);
    const bool kept = j < count;
    const float c = kept ? -a.lse[j] * kLog2e : -INFINITY, weight = !kept ? 0.f : a.weight ? a.weight[j] : a.scale.lift;
    grads_of<T>(a, acc, u, v0, j, c, weight, kept ? (int64_t)a.label[j] - a.v0 - v0 : -1, a.loss[j], 0, lane);
  }
}

__device__ __forceinline__ void end_parts(const CeArgs& a, acc_t& acc, const Result& r, int64_t rows, int wave, int lane) {
  const int h = lane >> 5;
  float* const to = a.parts + (r.split * rows + r.m * kTile + (wave >> 2) * 128 + 4 * h) * a.dcols + r.n * kTile +
                    (wave & 3) * 64 + (lane & 31);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (a.add) {
        float before[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) before[i] = to[(int64_t)row_of(t, i) * a.dcols + 32 * u];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][u][i] += before[i];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) to[(int64_t)row_of(t, i) * a.dcols + 32 * u] = acc[t][u][i];
      batch();
    }
}

template <typename T>
__device__ __forceinline__ void end_dw(const CeArgs& a, acc_t& acc, const Result& r, int wave, int lane) {
  const int h = lane >> 5, odd = lane & 1;
  const float f = a.scale();
  // lanes 2 k and 2 k + 1 swap, so that each has two neighbours of one row
  const int64_t v0 = a.v0 + r.m * kTile + (wave >> 2) * 128 + 4 * h + odd;
  const int d0 = r.n * kTile + (wave & 3) * 64 + (lane & 31) - odd;
  const int64_t left = a.vocab - v0;
  const bool even_rows = (a.dim & 1) == 0;
  uint8_t* const to = a.dw + 2 * (v0 * a.dim + d0);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float x = acc[t][u][i] * f, y = acc[t][u][i + 1] * f;
        const float give = odd ? x : y;
        const float take =
            __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(give), 0xB1, 0xF, 0xF, false));
        const uint32_t two = odd ? pack2<T>(take, y) : pack2<T>(x, take);
        const int d = d0 + 32 * u;
        if (row_of(t, i) < left && d < a.dim) {
          uint8_t* const at = to + 2 * ((int64_t)row_of(t, i) * a.dim + 32 * u);
          if (even_rows) {
            *(uint32_t*)at = two;
          } else {
            *(uint16_t*)at = (uint16_t)two;
            if (d + 1 < a.dim) *(uint16_t*)(at + 2) = (uint16_t)(two >> 16);
          }
        }
      }
      batch();
    }
}

template <typename T, Product P>
__global__ __launch_bounds__(kThreads, 2) void ce_product(const CeArgs a) {
  __shared__ __align__(1024) uint8_t smem[2 * kStage];
  lds_u8* const lds = (lds_u8*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = __builtin_amdgcn_readfirstlane(*a.count);
  const int chunks = (a.dim + 7) / 8, dpad = (int)(a.x_stride / 2);
  const int64_t entries = min((int64_t)a.piece, a.vocab - a.v0);  // of the piece
  const int token_tiles = (n + kTile - 1) / kTile, entry_tiles = (int)((entries + kTile - 1) / kTile),
            dim_tiles = a.dcols / kTile;
  const int token_steps = (n + kDepth - 1) / kDepth;
  const Order order =
      P == kLoss || P == kGrads ? Order(entry_tiles, token_tiles, dpad / kDepth, 1)
      : P == kDx ? Order(token_tiles, dim_tiles, (int)((entries + kDepth - 1) / kDepth),
                         splits_of(token_tiles, dim_tiles, a.piece / kDepth))
                 : Order(entry_tiles, dim_tiles, token_steps * (a.pair ? 2 : 1), a.splits);
  if constexpr (P == kDw) {
    if (n == 0 && a.splits == 1) {  // no token counts: zeros
      const int64_t first = a.v0 * a.dim, all = entries * a.dim;
      for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < all; i += (int64_t)gridDim.x * kThreads)
        ((uint16_t*)a.dw)[first + i] = 0;
      return;
    }
  }
  const uint8_t* const w = a.w + a.v0 * a.w_stride;

  Result run, ahead;  // the result in work, and the one whose tiles are loaded
  RowsTile ra, rb;
  ColsTile cb;
  const auto aim = [&]() {
    if constexpr (P == kLoss || P == kGrads) {
      ra.at(w, a.w_stride, (int64_t)ahead.m * kTile, entries, wave, lane);
      rb.at(a.x, a.x_stride, (int64_t)ahead.n * kTile, n, wave, lane);
    } else if constexpr (P == kDx) {
      cb.at(w, ahead.n * kTile, chunks, wave, lane);
    } else {
      cb.at(a.x, ahead.n * kTile, dpad / 8, wave, lane);
    }
  };
  // a wave's eight loads of a step, two steps ahead of the products
  int load_step;
  const auto load = [&](int stage, int part) {
    lds_u8* const to = lds + stage * kStage + (part >> 2) * kHalf;
    const int q = part & 3;
    if constexpr (P == kLoss || P == kGrads) {
      if (part < 4)
        ra.load(to, q, load_step, chunks, wave);
      else
        rb.load(to, q, load_step, dpad / 8, wave);
    } else if constexpr (P == kDx) {
      if (part < 4)
        load_tokens(a.d, to, q, load_step, ahead.m, a.npad, wave, lane);
      else
        cb.load(to, q, load_step, a.w_stride, entries, wave, lane);
    } else {
      if (part < 4)
        load_entries(a.d, to, q, load_step, ahead.m, a.npad, wave, lane);
      else
        cb.load(to, q, load_step < token_steps ? load_step : load_step - token_steps, a.x_stride, n, wave, lane);
    }
  };
  if (!ahead.next(order, true)) return;
  run = ahead;
  aim();
  load_step = ahead.k0;
  // on to the next step; behind the last one it is loaded again, which nobody reads, so that the loads need no branches
  const auto loaded = [&]() {
    if (load_step + 1 < ahead.k1) {
      ++load_step;
      return;
    }
    Result after = ahead;
    if (after.next(order, false)) {
      ahead = after;
      aim();
      load_step = ahead.k0;
    }
  };

  // this lane's place in the operands' tiles
  const uint32_t base = lds_address(lds);
  const uint32_t at_a = base + (P == kLoss || P == kGrads ? rows_lane(lane) + (wave >> 2) * 16384
                                : P == kDx                ? tokens_lane(lane) + (wave >> 2) * 4096
                                                          : entries_lane(lane) + (wave >> 2) * 16384);
  const uint32_t at_b = base + kHalf + (P == kLoss || P == kGrads ? rows_lane(lane) + (wave & 3) * 8192
                                                                  : cols_lane(lane) ^ (uint32_t)((wave & 3) * 128));
  frag_t fa[2][4], fb[2][2];
  const auto read = [&](int set, int stage, int s) {
    const uint32_t pa = at_a + stage * kStage, pb = at_b + stage * kStage;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      fb[set][u] = P == kLoss || P == kGrads ? rows_frag(pb, u, s) : cols_frag(pb, u, s);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      fa[set][t] = P == kLoss || P == kGrads ? rows_frag(pa, t, s) : P == kDx ? tokens_frag(pa, t, s) : entries_frag(pa, t, s);
  };
  acc_t acc = {};
  // with_each(t): between the products
  const auto multiply = [&](int set, auto with_each) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int u = 0; u < 2; ++u) acc[t][u] = mfma32<T>(fa[set][t], fb[set][u], acc[t][u]);
      keep_order();
      with_each(t);
    }
  };
  const auto nothing = [](int) {};

#pragma unroll
  for (int part = 0; part < 8; ++part) load(0, part);
  loaded();
#pragma unroll
  for (int part = 0; part < 4; ++part) load(1, part);
  tile_wait<4>();
  __syncthreads();
  read(0, 0, 0);
  for (int stage = 0, step = run.k0;; stage ^= 1) {
    read(1, stage, 1);
    keep_order();
    multiply(0, [&](int t) { load(stage ^ 1, 4 + t); });
    loaded();
    read(0, stage, 2);
    keep_order();
    multiply(1, nothing);
    read(1, stage, 3);
    keep_order();
    multiply(0, nothing);
    // every wave has read this stage and loaded the next
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const bool ends = ++step == run.k1;
    Result after = run;
    const bool last = ends && !after.next(order, false);
    if (!last) read(0, stage ^ 1, 0);
    keep_order();
    multiply(1, [&](int t) { load(stage, t); });
    if (ends) {
      if constexpr (P == kLoss) end_loss(a, acc, run, wave, lane);
      if constexpr (P == kGrads) end_grads<T>(a, acc, run, n, wave, lane);
      if constexpr (P == kDx) end_parts(a, acc, run, token_tiles * kTile, wave, lane);
      if constexpr (P == kDw) {
        if (a.splits > 1)
          end_parts(a, acc, run, a.piece, wave, lane);
        else
          end_dw<T>(a, acc, run, wave, lane);
      }
      if (last) {
        tile_wait<0>();  // no load may outlive the workgroup's LDS
        break;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) acc[t][u] = f32x16_t{};
      run = after;
      step = run.k0;
    }
  }
}

// ---------------------------------------------------------------------------
// The same product for few tokens, which reading weight once bounds (151936 x 1024 bf16, 64 tokens: 56 us, 5.6 TB/s, against
// 99 with ce_product's tiles; 128 tokens 87 against 99; more go there): tiles of 128 entries x 64 tokens by 8 waves (4 x 2, each
// 32 x 32), 64 deep, in a ring of five stages of 24 KB, four of which are on their way. What the epilogue reads of the
// tokens lies in LDS from the start: a load of its own would wait for the whole ring.
// ---------------------------------------------------------------------------
constexpr int kFew = 128;  // tokens
constexpr int kFewM = 128, kFewN = 64, kRing = 5, kFewStage = (kFewM + kFewN) * 128;

template <typename T, Product P>
__global__ __launch_bounds__(kThreads, 2) void ce_few(const CeArgs a) {
  static_assert(P == kLoss || P == kGrads, "the products with tokens for columns");
  __shared__ __align__(1024) uint8_t smem[kRing * kFewStage];
  __shared__ float ref_s[kFew], lse_s[kFew], weight_s[kFew];  // kGrads: ref_s is the loss
  __shared__ int32_t label_s[kFew];
  __shared__ float2 sum_s[kFewM / 32][kFewN];
  lds_u8* const lds = (lds_u8*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int n = __builtin_amdgcn_readfirstlane(*a.count);
  const int chunks = (a.dim + 7) / 8, dpad = (int)(a.x_stride / 2);
  const int64_t entries = min((int64_t)a.piece, a.vocab - a.v0);
  const Order order((int)((entries + kFewM - 1) / kFewM), (n + kFewN - 1) / kFewN, dpad / kDepth, 1);
  const uint8_t* const w = a.w + a.v0 * a.w_stride;
  Result run, ahead;
  if (!ahead.next(order, true)) return;
  run = ahead;
  if (tid < kFew) {
    const bool kept = tid < n;
    ref_s[tid] = P == kLoss ? a.ref[tid] : a.loss[tid];
    label_s[tid] = a.label[tid];
    if constexpr (P == kGrads) {
      lse_s[tid] = kept ? -a.lse[tid] * kLog2e : -INFINITY;
      weight_s[tid] = !kept ? 0.f : a.weight ? a.weight[tid] : a.scale.lift;
    }
  }
  RowsTile ra, rb;
  int load_step = ahead.k0;
  const auto aim = [&]() {
    ra.at(w, a.w_stride, (int64_t)ahead.m * kFewM, entries, wave, lane);
    rb.at(a.x, a.x_stride, (int64_t)ahead.n * kFewN, n, wave, lane);
  };
  const auto load_next = [&](int stage) {
    lds_u8* const to = lds + stage * kFewStage;
    ra.load(to, 0, load_step, chunks, wave);
    ra.load(to, 1, load_step, chunks, wave);
    rb.load(to + kFewM * 128, 0, load_step, dpad / 8, wave);
    if (load_step + 1 < ahead.k1) {
      ++load_step;
      return;
    }
    Result after = ahead;
    if (after.next(order, false)) {
      ahead = after;
      aim();
      load_step = ahead.k0;
    }
  };
  aim();
#pragma unroll
  for (int k = 0; k < kRing - 1; ++k) load_next(k);
  const uint32_t at_a = lds_address(lds) + rows_lane(lane) + (wave >> 1) * 4096;
  const uint32_t at_b = lds_address(lds) + kFewM * 128 + rows_lane(lane) + (wave & 1) * 4096;
  f32x16_t acc[1][1] = {};
  for (int stage = 0, step = run.k0;; stage = stage + 1 == kRing ? 0 : stage + 1) {
    tile_wait<3 * (kRing - 2)>();  // this step's three loads are in
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    load_next(stage == 0 ? kRing - 1 : stage - 1);  // where the step before lay
    frag_t fa[4], fb[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      fa[s] = rows_frag(at_a + stage * kFewStage, 0, s);
      fb[s] = rows_frag(at_b + stage * kFewStage, 0, s);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) acc[0][0] = mfma32<T>(fa[s], fb[s], acc[0][0]);
    if (++step != run.k1) continue;
    const int64_t v0 = (int64_t)run.m * kFewM + (wave >> 1) * 32;
    const int column = (wave & 1) * 32 + (lane & 31), j = run.n * kFewN + column;
    cut(acc, entries - v0, h);
    if constexpr (P == kLoss) {
      const float2 sum = sum_of(acc, 0, ref_s[j], (int)(label_s[j] - v0) - 4 * h, a.target + j);
      if (h == 0) sum_s[wave >> 1][column] = sum;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (tid < kFewN) {
        float2 all = sum_s[0][tid];
#pragma unroll
        for (int k = 1; k < kFewM / 32; ++k)
          if (sum_s[k][tid].y != 0.f) all = joined(all, sum_s[k][tid]);
        a.sums[(int64_t)run.m * a.npad + run.n * kFewN + tid] = all;
      }
    } else {
      grads_of<T>(a, acc, 0, v0, j, lse_s[j], weight_s[j], label_s[j] < 0 ? -1 : label_s[j] - a.v0 - v0, ref_s[j],
                  (int64_t)order.n * kFewN / 32 * 1024, lane);
    }
    acc[0][0] = f32x16_t{};
    if (!run.next(order, false)) break;
    step = run.k0;
  }
  tile_wait<0>();  // no load may outlive the workgroup's LDS
}

// ---------------------------------------------------------------------------
// Around the products
// ---------------------------------------------------------------------------
constexpr int kPrepareRows = 16;  // tokens of a workgroup of ce_prepare, a wave each
constexpr int kCounted = 1024;    // of one of ce_count
// Tokens up to which ce_prepare counts alone: all of the forward with 256 entries, 64 wide, 28 us so and 28 to 30 with ce_count at 8192
// tokens, 39 and 37 at 16384; 152 and 91 at 65536, 18700 and 1250 at 2^20.
constexpr int64_t kFewToCount = 12288;
constexpr int kJoinTokens = 32, kJoinSlices = 32;

struct Header {
  int32_t count;   // kept tokens
  uint32_t ended;  // workgroups of ce_join that are done
};

template <typename L>
__device__ __forceinline__ int label_of(const void* labels, int64_t i, int64_t ignore, int64_t vocab) {
  const int64_t y = (int64_t)((const L*)labels)[i];
  return y == ignore || y < 0 || y >= vocab ? -1 : (int)y;
}

// Kept tokens of 1024 each: what ce_prepare counts from where a count of all labels before would be too long.
template <typename L>
__global__ __launch_bounds__(kCounted) void ce_count(const void* labels, int64_t tokens, int64_t ignore, int64_t vocab,
                                                     int32_t* counts) {
  const int64_t i = (int64_t)blockIdx.x * kCounted + threadIdx.x;
  const int n = __syncthreads_count(i < tokens && label_of<L>(labels, i, ignore, vocab) >= 0);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

constexpr int kNothing = -1000;  // the exponent of a row of zeros

// The kept tokens side by side: rows, labels, places, and the label's logit; in f16 the exponent of a row's largest number. A
// workgroup counts the kept tokens before its 16 itself: 16384 tokens' labels are read 512 times in all, 67 MB out of the L2,
// and no launch is needed to count. For more tokens, whose square that grows with, from ce_count's sums of 1024.
template <typename T, typename L>
__global__ __launch_bounds__(1024) void ce_prepare(const T* __restrict__ x, int64_t x_stride, int64_t tokens,
                                                   const T* __restrict__ w, int64_t w_stride, int64_t vocab, int dim, int dpad,
                                                   int wide, const void* labels, int64_t ignore, Header* head, int32_t* place,
                                                   int32_t* token, int32_t* label, float* ref, int32_t* size, T* __restrict__ kept,
                                                   int npad, float* losses, const int32_t* __restrict__ counts) {
  __shared__ int32_t before_s[16], own_s[16];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int64_t first = (int64_t)blockIdx.x * kPrepareRows, i = first + wave;
  const int y = i < tokens ? label_of<L>(labels, i, ignore, vocab) : -1;
  int32_t before = 0;
  const int64_t whole = counts ? first / kCounted : 0;
  for (int64_t k = tid; k < whole; k += 1024) before += counts[k];
  for (int64_t k = whole * kCounted + tid; k < first; k += 1024) before += label_of<L>(labels, k, ignore, vocab) >= 0;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) before += __shfl_xor(before, s);
  if (lane == 0) {
    before_s[wave] = before;
    own_s[wave] = y >= 0;
  }
  __syncthreads();
  int at = 0, own = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    at += before_s[k];
    own += own_s[k];
  }
  const int count = at + own;  // with this workgroup's
#pragma unroll
  for (int k = 0; k < 16; ++k) at += k < wave ? own_s[k] : 0;
  if (blockIdx.x == gridDim.x - 1) {
    if (tid == 0) {
      head->count = count;
      head->ended = 0;
    }
    for (int j = count + tid; j < npad; j += 1024) {
      label[j] = -1;
      ref[j] = 0.f;
    }
  }
  if (i >= tokens) return;
  if (lane == 0) {
    place[i] = y >= 0 ? at : -1;
    if (y >= 0) {
      token[at] = (int)i;
      label[at] = y;
    } else if (losses) {
      losses[i] = 0.f;
    }
  }
  if (y < 0) return;
  const T* const row = x + i * x_stride;
  T* const to = kept + (int64_t)at * dpad;
  const T* const wy = w + (int64_t)y * w_stride;
  float dot = 0.f;
  int top = 0;  // bits of the largest finite number's size, f16
  const auto measure = [&](uint32_t bits) {
    const int a = (int)(bits & 0x7fffu);
    if (a < 0x7c00) top = max(top, a);
  };
  if (wide) {
    for (int c = lane; c < dpad / 8; c += 64) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (c < dim / 8) {
        v = ld16(row + 8 * c);
        dot = vec_dot<T>(v, ld16(wy + 8 * c), dot);
        if constexpr (__is_same(T, f16_t)) {
#pragma unroll
          for (const uint32_t two : {v.x, v.y, v.z, v.w}) {
            measure(two);
            measure(two >> 16);
          }
        }
      }
      st16(to + 8 * c, v);
    }
  } else {
    for (int c = lane; c < dpad; c += 64) {
      uint16_t v = 0;
      if (c < dim) {
        v = ((const uint16_t*)row)[c];
        dot += unpack1<T>(v) * unpack1<T>(((const uint16_t*)wy)[c]);
        measure(v);
      }
      ((uint16_t*)to)[c] = v;
    }
  }
  dot = group_sum<64>(dot);
  if (lane == 0) ref[at] = dot;
  if constexpr (__is_same(T, f16_t)) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = max(top, __shfl_xor(top, s));
    if (lane == 0) size[at] = top == 0 ? kNothing : __builtin_amdgcn_frexp_expf(unpack1<T>((uint32_t)top));
  }
}

// lse and loss of 32 tokens from the tiles' sums. losses: one for each token. mean: else the workgroup that ends last adds
// all workgroups' losses, in order.
__global__ __launch_bounds__(kJoinTokens* kJoinSlices) void ce_join(Header* head, const float2* __restrict__ sums, int parts,
                                                                    int npad, const float* __restrict__ target,
                                                                    const int32_t* __restrict__ token, float* __restrict__ lse,
                                                                    float* __restrict__ own_loss,
                                                                    float* losses, float* block_sums, float* total, int mean) {
  __shared__ float2 s[kJoinSlices][kJoinTokens];
  __shared__ float sum_s[kJoinSlices / 2];
  __shared__ bool ends_s;
  const int t = threadIdx.x % kJoinTokens, slice = threadIdx.x / kJoinTokens;
  const int j = blockIdx.x * kJoinTokens + t, count = head->count;
  float m = -INFINITY, sum = 0.f;
  const auto add = [&](float r, float v) {
    const float2 both = joined(make_float2(m, sum), make_float2(r, v));  // 0 at first
    m = both.x;
    sum = both.y;
  };
  if (j < count) {
    constexpr int FLIGHT = 8;
    for (int p = slice; p < parts; p += kJoinSlices * FLIGHT) {
      float2 v[FLIGHT];
#pragma unroll
      for (int k = 0; k < FLIGHT; ++k) v[k] = sums[(int64_t)min(p + k * kJoinSlices, parts - 1) * npad + j];
#pragma unroll
      for (int k = 0; k < FLIGHT; ++k)
        if (p + k * kJoinSlices < parts) add(v[k].x, v[k].y);
    }
  }
  s[slice][t] = make_float2(m, sum);
  __syncthreads();
  if (slice == 0) {
    float loss = 0.f;
    if (j < count) {
      for (int k = 1; k < kJoinSlices; ++k)
        if (s[k][t].y != 0.f) add(s[k][t].x, s[k][t].y);  // NaN counts as something
      // log(1 + the others' exponentials against the label's), for exponents of any size
      const float z = target[j], x = logf(sum) + (m - z);
      loss = fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)));
      if (x != x) loss = x;
      lse[j] = loss < INFINITY ? z + loss : m + logf(sum);
      own_loss[j] = loss;
      if (losses) losses[token[j]] = loss;
    }
#pragma unroll
    for (int k = 1; k < kJoinTokens; k <<= 1) loss += __shfl_xor(loss, k);
    if (t == 0 && !losses) {
      __hip_atomic_store(&block_sums[blockIdx.x], loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      ends_s = __hip_atomic_fetch_add(&head->ended, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
  }
  if (losses) return;
  __syncthreads();
  if (!ends_s) return;
  sum = 0.f;
  for (int k = threadIdx.x; k < (int)gridDim.x; k += kJoinTokens * kJoinSlices)
    sum += __hip_atomic_load(&block_sums[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  sum = group_sum<64>(sum);
  if ((threadIdx.x & 63) == 0) sum_s[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = 0.f;
  for (int k = 0; k < kJoinSlices / 2; ++k) sum += sum_s[k];
  *total = mean ? sum / (float)max(count, 1) : sum;
}

// The tokens' gradients as weights of d, in bf16: g_j over a power of two that the largest is just below; the results' scale
// undoes it. One gradient for all tokens is a scale alone: nothing is weighted then, and neither this nor ce_units runs.
__global__ __launch_bounds__(1024) void ce_weights(float* scale, const float* __restrict__ grad, const int32_t* __restrict__ place,
                                                   int64_t tokens, float* __restrict__ weight) {
  __shared__ float s[16];
  const int tid = threadIdx.x;
  float top = 0.f;
  for (int64_t i = tid; i < tokens; i += 1024)
    if (place[i] >= 0) top = fmaxf(top, fabsf(grad[i]));
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
  if ((tid & 63) == 0) s[tid >> 6] = top;
  __syncthreads();
  for (int k = 0; k < 16; ++k) top = fmaxf(top, s[k]);
  const int e = top > 0.f ? min(max(__builtin_amdgcn_frexp_expf(top), -100), 100) : 0;
  const float unit = ldexpf(1.f, e);
  for (int64_t i = tid; i < tokens; i += 1024)
    if (place[i] >= 0) weight[place[i]] = grad[i] / unit;
  if (tid == 0) *scale = unit;
}

// The same in f16, whose range one power of two does not do for: each token's d is held in units of its own gradient, with
// its largest numbers near `lift` = 2^14 (its softmax weights reach f16's smallest). dx's rows are scaled one by one (unit). dW
// sums over tokens: their powers of two go to a copy of the hidden states for that product (ce_scaled), in which the largest
// product of a gradient and a state is just below 2^15, so that those down to 2^-29 of it keep their precision. (One power
// for all rounded the d of gradients far below the largest away: 2^-24 of it, a softmax of 32000 entries, were zeros.)
__global__ __launch_bounds__(1024) void ce_units(float* scale, const float* __restrict__ grad, const int32_t* __restrict__ place,
                                                 int64_t tokens, float lift, const int32_t* __restrict__ size,
                                                 float* __restrict__ weight, float* __restrict__ unit, float* __restrict__ factor) {
  __shared__ int32_t s[16];
  const int tid = threadIdx.x;
  const auto exponent = [](float g) { return min(max(__builtin_amdgcn_frexp_expf(g), -100), 100); };
  int top = kNothing;
  for (int64_t i = tid; i < tokens; i += 1024) {
    const int j = place[i];
    if (j < 0) continue;
    const float g = grad[i];
    const bool finite = fabsf(g) < INFINITY;
    const int e = finite && g != 0.f ? exponent(g) : 0;
    weight[j] = ldexpf(g, -e) * lift;
    unit[j] = ldexpf(1.f, e) / lift;
    if (finite && g != 0.f && size[j] != kNothing) top = max(top, e + size[j]);
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) top = max(top, __shfl_xor(top, k));
  if ((tid & 63) == 0) s[tid >> 6] = top;
  __syncthreads();
  for (int k = 0; k < 16; ++k) top = max(top, s[k]);
  if (top == kNothing) top = 0;
  for (int64_t i = tid; i < tokens; i += 1024) {
    const int j = place[i];
    if (j < 0) continue;
    const float g = grad[i];
    // a gradient of 0 has no part in `top`: its states, which count for nothing, are not to overflow
    const int e = g == 0.f ? -1000 : fabsf(g) < INFINITY ? exponent(g) : 0;
    factor[j] = ldexpf(1.f, min(max(e + 15 - top, -126), 126));
  }
  if (tid == 0) *scale = ldexpf(1.f, top - 15) / lift;
}

// The kept tokens' hidden states times their powers of two, f16, a wave a row.
__global__ __launch_bounds__(256) void ce_scaled(const int32_t* count, const uint8_t* __restrict__ x, const float* __restrict__ factor,
                                                 int dpad, uint8_t* __restrict__ out) {
  const int lane = threadIdx.x & 63, n = *count;
  for (int64_t j = blockIdx.x * 4 + (threadIdx.x >> 6); j < n; j += gridDim.x * 4) {
    const float by = factor[j];
    for (int c = lane; c < dpad / 8; c += 64) {
      const int64_t at = (j * dpad + 8 * c) * 2;
      float f[8];
      VecTraits<f16_t>::unpack(ld16(x + at), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= by;
      st16(out + at, VecTraits<f16_t>::pack(f));
    }
  }
}

// What rounding left of the label's d, the one large number among a token's.
template <typename T>
__device__ __forceinline__ float label_rest(const CeArgs& a, int64_t j) {
  const float x = label_d(a.loss[j], a.weight ? a.weight[j] : a.scale.lift);
  return x - unpack1<T>(pack2<T>(x, x) & 0xffffu);
}

// Rows of results: the splits' sums in order, scaled and rounded, a workgroup a row at a time. dx (place): row i from row
// place[i], zeros if that is negative, with what the rounding left of d: of all of it from a row of its own (pair), else of
// the label's times its row of the weight; `splits` is 0, the kept tokens give it. dW (place NULL): row i from row i; few kept
// tokens leave some splits without a step, which wrote nothing.
template <typename T>
__global__ __launch_bounds__(256) void ce_rows(const CeArgs a, const int32_t* __restrict__ place, int64_t rows,
                                               const float* __restrict__ parts, int splits, T* __restrict__ out) {
  const float all = a.scale();
  const int n = *a.count, tiles = (n + kTile - 1) / kTile, steps = (n + kDepth - 1) / kDepth, dim = a.dim;
  int64_t pad = a.piece;
  if (place) {
    splits = splits_of(tiles, a.dcols / kTile, a.piece / kDepth);
    pad = tiles * kTile;
  }
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    const int64_t j = place ? place[i] : i;
    const float rest = place && j >= 0 && !a.pair ? label_rest<T>(a, j) : 0.f;
    const float f = place && j >= 0 && a.unit ? a.unit[j] : all;
    const uint8_t* const wy = a.w + (place && j >= 0 ? a.label[j] * a.w_stride : 0);
    for (int d = threadIdx.x * 4; d < dim; d += 1024) {
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      const auto add = [&](int s, int64_t row) {
        const float4 v = *(const float4*)(parts + (s * pad + row) * a.dcols + d);
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      };
      if (place && j >= 0) {
#pragma unroll 8
        for (int s = 0; s < splits; ++s) add(s, j);
        if (a.pair)
          for (int s = 0; s < splits; ++s) add(s, j + steps * kDepth);
        const uint2 y = *(const uint2*)(wy + 2 * d);  // rows reach to a multiple of 8
        sum.x = __builtin_fmaf(rest, unpack1<T>(y.x & 0xffffu), sum.x);
        sum.y = __builtin_fmaf(rest, unpack1<T>(y.x >> 16), sum.y);
        sum.z = __builtin_fmaf(rest, unpack1<T>(y.y & 0xffffu), sum.z);
        sum.w = __builtin_fmaf(rest, unpack1<T>(y.y >> 16), sum.w);
      } else if (!place) {
        for (int s = 0; s < splits; ++s)
          if ((int64_t)steps * s / splits < (int64_t)steps * (s + 1) / splits) add(s, j);
      }
      uint16_t* const to = (uint16_t*)(out + i * dim + d);
      const uint32_t p = j < 0 ? 0u : pack2<T>(sum.x * f, sum.y * f), q = j < 0 ? 0u : pack2<T>(sum.z * f, sum.w * f);
      if ((dim & 3) == 0) {
        *(uint2*)to = make_uint2(p, q);
      } else {
        const uint16_t four[4] = {(uint16_t)p, (uint16_t)(p >> 16), (uint16_t)q, (uint16_t)(q >> 16)};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (d + k < dim) to[k] = four[k];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// What the forward leaves for the backward, in one buffer.
struct Kept {
  int64_t npad, dpad, place, token, label, ref, target, lse, loss, size, x, bytes;
};
bool plan_kept(int64_t tokens, int64_t dim, Kept* k) {
  if (tokens < 0 || dim < 1 || tokens >= (1ll << 22) || dim > 65536) return false;
  k->npad = up(tokens < 1 ? 1 : tokens, kTile);
  k->dpad = up(dim, kDepth);
  k->place = 256;
  k->token = k->place + k->npad * 4;
  k->label = k->token + k->npad * 4;
  k->ref = k->label + k->npad * 4;
  k->target = k->ref + k->npad * 4;
  k->lse = k->target + k->npad * 4;
  k->loss = k->lse + k->npad * 4;
  k->size = k->loss + k->npad * 4;
  k->x = k->size + k->npad * 4;
  k->bytes = k->x + k->npad * k->dpad * 2;
  return true;
}

struct Forward {
  int64_t sums, block_sums, counts, bytes;
};
Forward plan_forward(const Kept& k, int64_t vocab) {
  Forward f;
  f.sums = 0;
  f.block_sums = f.sums + up(vocab, kTile) / 128 * k.npad * 8;
  f.counts = f.block_sums + k.npad / kJoinTokens * 4;
  f.bytes = f.counts + up(k.npad, kCounted) / kCounted * 4;
  return f;
}

struct Backward {
  int64_t piece, dcols, dw_splits, weight, unit, factor, scaled, d, dx, dw, bytes;
};
Backward plan_backward(const Kept& k, int64_t vocab, int64_t dim) {
  Backward b;
  const int64_t all = up(vocab, kTile) / kTile, tokens = k.npad / kTile;
  // 768 MB of d at a time at most, and no fewer than 64 tiles of the vocabulary: dW's product has one for each and 256 columns
  int64_t most = 3 * (1ll << 27) / k.npad / kTile;
  if (most < 64) most = 64;
  // Of the fewest pieces and a few more, those whose products leave the fewest workgroups idle in their last rounds
  // (2048 tokens, 151936 entries: one piece of 594 tiles 19 + 10 rounds, two of 297 20 + 10; 16384 tokens: ten pieces)
  const auto rounds = [&](int64_t tiles) {
    const auto of = [](int64_t m, int64_t n) { return (Blocks(m, n).results() + 255) / 256; };
    return of(tiles, tokens) * (k.dpad / kDepth + 2) + of(tiles, up(dim, kTile) / kTile) * (k.npad / kDepth + 2);
  };
  const int64_t fewest = (all + most - 1) / most;
  int64_t best = 0, pieces = fewest;
  for (int64_t n = fewest; n <= fewest + 4 && n <= all; ++n) {
    const int64_t tiles = (all + n - 1) / n, whole = all / tiles;
    const int64_t cost = whole * rounds(tiles) + (all > whole * tiles ? rounds(all - whole * tiles) : 0);
    if (best == 0 || cost < best) {
      best = cost;
      pieces = n;
    }
  }
  b.piece = (all + pieces - 1) / pieces * kTile;
  b.dcols = up(dim, kTile);
  const int64_t cols = b.dcols / kTile;
  b.dw_splits = b.piece < vocab ? 1 : splits_of(b.piece / kTile, cols, k.npad / kDepth);
  b.weight = 256;  // behind the results' scale
  b.unit = b.weight + k.npad * 4;
  b.factor = b.unit + k.npad * 4;
  b.scaled = b.factor + k.npad * 4;
  b.d = b.scaled + k.npad * k.dpad * 2;
  b.dx = b.d + b.piece * k.npad * 2;
  // dx's sum is split by the kept tokens, whose number the device has: splits x tiles of tokens are 256 / cols or fewer where
  // there are several splits, and no more than the steps allow
  const int64_t tiles = k.npad / kTile, most_splits = splits_of(1, 1, b.piece / kDepth);
  int64_t parts = tiles * most_splits < 256 / cols ? tiles * most_splits : 256 / cols;
  if (parts < tiles) parts = tiles;
  b.dw = b.dx + parts * kTile * b.dcols * 4;
  b.bytes = b.dw + (b.dw_splits > 1 ? b.dw_splits * b.piece * b.dcols * 4 : 0);
  return b;
}

template <typename T, Product P>
void launch(const CeArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((ce_product<T, P>), dim3(256), dim3(kThreads), 0, st, a);
}

template <typename T, Product P>
void launch_logits(const CeArgs& a, int64_t tokens, hipStream_t st) {
  if (tokens <= kFew)
    hipLaunchKernelGGL((ce_few<T, P>), dim3(256), dim3(kThreads), 0, st, a);
  else
    launch<T, P>(a, st);
}

template <typename T>
int run_forward(const void* x, int64_t x_stride, int64_t tokens, const void* w, int64_t w_stride, int64_t vocab, int64_t dim,
                const void* labels, int bits, int64_t ignore, int reduction, float* loss, uint8_t* kept, const Kept& k, uint8_t* ws,
                const Forward& f, hipStream_t st) {
  Header* const head = (Header*)kept;
  int32_t *place = (int32_t*)(kept + k.place), *token = (int32_t*)(kept + k.token), *label = (int32_t*)(kept + k.label);
  float *ref = (float*)(kept + k.ref), *target = (float*)(kept + k.target), *lse = (float*)(kept + k.lse);
  float* const losses = reduction == 0 ? loss : nullptr;
  const int wide = (((uintptr_t)x | (uintptr_t)w) & 15) == 0 && ((x_stride | w_stride | dim) & 7) == 0;
  const unsigned blocks = (unsigned)((tokens < 1 ? 1 : tokens) + kPrepareRows - 1) / kPrepareRows;
  int32_t* const counts = tokens > kFewToCount ? (int32_t*)(ws + f.counts) : nullptr;
  const dim3 counted((unsigned)((tokens + kCounted - 1) / kCounted));
  if (counts && bits == 64)
    hipLaunchKernelGGL((ce_count<int64_t>), counted, dim3(kCounted), 0, st, labels, tokens, ignore, vocab, counts);
  else if (counts)
    hipLaunchKernelGGL((ce_count<int32_t>), counted, dim3(kCounted), 0, st, labels, tokens, ignore, vocab, counts);
  if (bits == 64)
    hipLaunchKernelGGL((ce_prepare<T, int64_t>), dim3(blocks), dim3(1024), 0, st, (const T*)x, x_stride, tokens, (const T*)w,
                       w_stride, vocab, (int)dim, (int)k.dpad, wide, labels, ignore, head, place, token, label, ref,
                       (int32_t*)(kept + k.size), (T*)(kept + k.x), (int)k.npad, losses, counts);
  else
    hipLaunchKernelGGL((ce_prepare<T, int32_t>), dim3(blocks), dim3(1024), 0, st, (const T*)x, x_stride, tokens, (const T*)w,
                       w_stride, vocab, (int)dim, (int)k.dpad, wide, labels, ignore, head, place, token, label, ref,
                       (int32_t*)(kept + k.size), (T*)(kept + k.x), (int)k.npad, losses, counts);
  CeArgs a = {};
  a.x = kept + k.x;
  a.x_stride = k.dpad * 2;
  a.w = (const uint8_t*)w;
  a.w_stride = w_stride * 2;
  a.count = &head->count;
  a.label = label;
  a.ref = ref;
  a.target = target;
  a.sums = (float2*)(ws + f.sums);
  a.vocab = vocab;
  a.piece = (int32_t)up(vocab, kTile);
  a.dim = (int32_t)dim;
  a.npad = (int32_t)k.npad;
  a.dcols = (int32_t)up(dim, kTile);
  a.splits = 1;
  launch_logits<T, kLoss>(a, tokens, st);
  const int64_t joins = (tokens < 1 ? 1 : tokens) + kJoinTokens - 1;
  if (reduction == 0 && tokens == 0) return pkm_check_launch("pkm_linear_ce_fwd");  // no loss to write
  hipLaunchKernelGGL(ce_join, dim3((unsigned)(joins / kJoinTokens)), dim3(kJoinTokens * kJoinSlices), 0, st, head,
                     (const float2*)a.sums, (int)((vocab + 127) / 128), (int)k.npad, target, token, lse,
                     (float*)(kept + k.loss), losses, (float*)(ws + f.block_sums), loss, reduction == 1);
  return pkm_check_launch("pkm_linear_ce_fwd");
}

template <typename T>
int run_backward(const uint8_t* kept, const Kept& k, int64_t tokens, const void* w, int64_t w_stride, int64_t vocab, int64_t dim,
                 const float* grad, int reduction, void* dx, void* dw, uint8_t* ws, const Backward& b, hipStream_t st) {
  const Header* const head = (const Header*)kept;
  const int32_t* place = (const int32_t*)(kept + k.place);
  constexpr bool half = __is_same(T, f16_t);
  constexpr float lift = half ? 16384.f : 1.f;
  CeArgs a = {};
  const uint8_t* dw_x = kept + k.x;
  if (reduction == 0) {
    float* weight = (float*)(ws + b.weight);
    a.weight = weight;
    if constexpr (half) {
      float *unit = (float*)(ws + b.unit), *factor = (float*)(ws + b.factor);
      a.unit = unit;
      hipLaunchKernelGGL(ce_units, dim3(1), dim3(1024), 0, st, (float*)ws, grad, place, tokens, lift,
                         (const int32_t*)(kept + k.size), weight, unit, factor);
      if (dw) {
        dw_x = ws + b.scaled;
        const int64_t blocks = (tokens + 3) / 4;
        if (blocks > 0)
          hipLaunchKernelGGL(ce_scaled, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, &head->count,
                             kept + k.x, factor, (int)k.dpad, ws + b.scaled);
      }
    } else {
      hipLaunchKernelGGL(ce_weights, dim3(1), dim3(1024), 0, st, (float*)ws, grad, place, tokens, weight);
    }
  }
  a.x_stride = k.dpad * 2;
  a.w = (const uint8_t*)w;
  a.w_stride = w_stride * 2;
  a.d = ws + b.d;
  a.count = &head->count;
  a.label = (const int32_t*)(kept + k.label);
  a.loss = (const float*)(kept + k.loss);
  a.lse = (const float*)(kept + k.lse);
  a.dw = (uint8_t*)dw;
  a.scale = Scale{(const float*)ws, reduction == 0 ? nullptr : grad, &head->count, lift, reduction == 1};
  a.vocab = vocab;
  a.piece = (int32_t)b.piece;
  a.dim = (int32_t)dim;
  a.npad = (int32_t)k.npad;
  a.dcols = (int32_t)b.dcols;
  a.pair = tokens <= kFew;
  float *dx_parts = (float*)(ws + b.dx), *dw_parts = (float*)(ws + b.dw);
  for (int64_t v0 = 0; v0 < vocab; v0 += b.piece) {
    a.v0 = v0;
    a.x = kept + k.x;
    a.splits = 1;
    a.add = 0;
    launch_logits<T, kGrads>(a, tokens, st);
    if (dw) {
      a.x = dw_x;
      a.splits = (int32_t)b.dw_splits;
      a.parts = dw_parts;
      launch<T, kDw>(a, st);
    }
    if (dx) {
      a.parts = dx_parts;
      a.add = v0 > 0;
      launch<T, kDx>(a, st);
    }
  }
  const auto rows = [&](const int32_t* from, int64_t n, const float* parts, int64_t splits, void* out) {
    hipLaunchKernelGGL(ce_rows<T>, dim3((unsigned)(n < 65536 ? n : 65536)), dim3(256), 0, st, a, from, n, parts, (int)splits,
                       (T*)out);
  };
  if (dx && tokens > 0) rows(place, tokens, dx_parts, 0, dx);
  if (dw && b.dw_splits > 1) rows(nullptr, vocab, dw_parts, b.dw_splits, dw);
  return pkm_check_launch("pkm_linear_ce_bwd");
}

}  // namespace
}  // namespace pkm

using namespace pkm;

#define CE_REQUIRE_COMMON(fn)                                                                                               \
  PKM_REQUIRE(tokens >= 0 && vocab >= 1 && dim >= 1, PKM_ERR_INVALID_ARGUMENT, fn ": %lld tokens, weight [%lld, %lld]",     \
              (long long)tokens, (long long)vocab, (long long)dim);                                                         \
  PKM_REQUIRE(dtype == PKM_DTYPE_BF16 || dtype == PKM_DTYPE_F16, PKM_ERR_UNSUPPORTED,                                       \
              fn ": dtype %d not supported (bfloat16, float16 are)", dtype);                                                \
  PKM_REQUIRE(tokens < (1ll << 22) && dim <= 65536 && vocab < (1ll << 30), PKM_ERR_UNSUPPORTED,                             \
              fn ": %lld tokens, weight [%lld, %lld] (fewer than 2^22, 2^30, up to 65536 are supported)", (long long)tokens, \
              (long long)vocab, (long long)dim);                                                                            \
  PKM_REQUIRE(reduction >= 0 && reduction <= 2, PKM_ERR_INVALID_ARGUMENT, fn ": reduction %d", reduction);                  \
  Kept k;                                                                                                                   \
  plan_kept(tokens, dim, &k);                                                                                               \
  PKM_REQUIRE((up(vocab, kTile) / kTile + 32) * (k.npad / kTile + 32) < (1ll << 30), PKM_ERR_UNSUPPORTED,                   \
              fn ": %lld tokens of %lld entries are too many", (long long)tokens, (long long)vocab);                        \
  PKM_REQUIRE(weight && (((uintptr_t)weight) & 15) == 0 && (w_stride & 7) == 0 && w_stride >= up(dim, 8) &&                 \
                  w_stride <= (1ll << 22),                                                                                  \
              PKM_ERR_INVALID_ARGUMENT, fn ": weight has to lie on 16 bytes, its rows a multiple of 8 numbers apart");      \
  PKM_REQUIRE(kept && (((uintptr_t)kept) & 15) == 0 && kept_bytes >= (size_t)k.bytes, PKM_ERR_WORKSPACE,                    \
              fn ": kept buffer of %zu bytes, %lld needed", kept_bytes, (long long)k.bytes)

extern "C" size_t pkm_linear_ce_kept_size(int64_t tokens, int64_t dim) {
  Kept k;
  return plan_kept(tokens, dim, &k) ? (size_t)k.bytes : 0;
}

extern "C" size_t pkm_linear_ce_fwd_workspace_size(int64_t tokens, int64_t vocab, int64_t dim) {
  Kept k;
  return vocab >= 1 && vocab < (1ll << 30) && plan_kept(tokens, dim, &k) ? (size_t)plan_forward(k, vocab).bytes : 0;
}

extern "C" size_t pkm_linear_ce_bwd_workspace_size(int64_t tokens, int64_t vocab, int64_t dim) {
  Kept k;
  return vocab >= 1 && vocab < (1ll << 30) && plan_kept(tokens, dim, &k) ? (size_t)plan_backward(k, vocab, dim).bytes : 0;
}

extern "C" int pkm_linear_ce_fwd(const void* x, int64_t x_stride, int64_t tokens, const void* weight, int64_t w_stride,
                                 int64_t vocab, int64_t dim, int dtype, const void* labels, int label_bits, int64_t ignore,
                                 int reduction, float* loss, void* kept, size_t kept_bytes, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  CE_REQUIRE_COMMON("pkm_linear_ce_fwd");
  PKM_REQUIRE(label_bits == 32 || label_bits == 64, PKM_ERR_INVALID_ARGUMENT, "pkm_linear_ce_fwd: labels of %d bits (32 or 64)",
              label_bits);
  PKM_REQUIRE(tokens == 0 || (x && labels), PKM_ERR_INVALID_ARGUMENT, "pkm_linear_ce_fwd: null pointer");
  PKM_REQUIRE(loss || (tokens == 0 && reduction == 0), PKM_ERR_INVALID_ARGUMENT, "pkm_linear_ce_fwd: null pointer");
  PKM_REQUIRE(x_stride >= 0 && x_stride < (1ll << 40), PKM_ERR_INVALID_ARGUMENT, "pkm_linear_ce_fwd: row stride %lld",
              (long long)x_stride);
  const Forward f = plan_forward(k, vocab);
  PKM_REQUIRE(workspace && (((uintptr_t)workspace) & 15) == 0 && workspace_bytes >= (size_t)f.bytes, PKM_ERR_WORKSPACE,
              "pkm_linear_ce_fwd: workspace of %zu bytes, %lld needed", workspace_bytes, (long long)f.bytes);
  return dtype == PKM_DTYPE_BF16
             ? run_forward<bf16_t>(x, x_stride, tokens, weight, w_stride, vocab, dim, labels, label_bits, ignore, reduction,
                                   loss, (uint8_t*)kept, k, (uint8_t*)workspace, f, (hipStream_t)stream)
             : run_forward<f16_t>(x, x_stride, tokens, weight, w_stride, vocab, dim, labels, label_bits, ignore, reduction,
                                  loss, (uint8_t*)kept, k, (uint8_t*)workspace, f, (hipStream_t)stream);
}

extern "C" int pkm_linear_ce_bwd(const void* kept, size_t kept_bytes, int64_t tokens, const void* weight, int64_t w_stride,
                                 int64_t vocab, int64_t dim, int dtype, const float* grad_loss, int reduction, void* dx,
                                 void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  CE_REQUIRE_COMMON("pkm_linear_ce_bwd");
  PKM_REQUIRE(grad_loss || (tokens == 0 && reduction == 0), PKM_ERR_INVALID_ARGUMENT, "pkm_linear_ce_bwd: null pointer");
  PKM_REQUIRE((((uintptr_t)dx | (uintptr_t)dweight) & 15) == 0, PKM_ERR_INVALID_ARGUMENT,
              "pkm_linear_ce_bwd: dx and dweight have to lie on 16 bytes");
  const Backward b = plan_backward(k, vocab, dim);
  PKM_REQUIRE(workspace && (((uintptr_t)workspace) & 15) == 0 && workspace_bytes >= (size_t)b.bytes, PKM_ERR_WORKSPACE,
              "pkm_linear_ce_bwd: workspace of %zu bytes, %lld needed", workspace_bytes, (long long)b.bytes);
  return dtype == PKM_DTYPE_BF16
             ? run_backward<bf16_t>((const uint8_t*)kept, k, tokens, weight, w_stride, vocab, dim, grad_loss, reduction, dx,
                                    dweight, (uint8_t*)workspace, b, (hipStream_t)stream)
             : run_backward<f16_t>((const uint8_t*)kept, k, tokens, weight, w_stride, vocab, dim, grad_loss, reduction, dx, dweight,
                                   (uint8_t*)workspace, b, (hipStream_t)stream);
}
