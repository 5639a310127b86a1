// A paged key / value cache of 4-bit codes: written (quantised), read back,
// and attended over.
//
// A head vector of D numbers is held in groups of 32: minimum m, step
// s = (max - min) / 15 in the cache's type, codes c = round((x - m) / s); the number
// read back is m + s c. Number d = w + 16 i (w < 16) of a vector lies in its
// word w, D = 128: 32-bit words, bits 4 (i / 2 + 4 (i % 2)); D = 64: 16-bit words, bits 4 i.
// So one shift and one mask of a word give numbers of one group in both halves
// of a register, as the matrix instructions take them.
//   codes  [2 (K, V), pages, heads, page, D / 2] bytes
//   params [2 (K, V), pages, heads, 2 (s, m), D / 32, page] of the cache's type
// Position t of sequence b lies in page table[b, t / page], slot t % page.
#include "attn_common.h"

namespace pkm {
namespace {

constexpr int kThreads = 256;

struct Cache {
  uint8_t* codes;
  uint8_t* params;
  int64_t pages;
  int heads, page;
};

// Bytes from the start of codes / params to a page's head.
template <int D>
__device__ __forceinline__ int64_t codes_at(const Cache& c, int side, int page, int head) {
  return (((int64_t)side * c.pages + page) * c.heads + head) * c.page * (D / 2);
}
template <int D>
__device__ __forceinline__ int64_t params_at(const Cache& c, int side, int page, int head) {
  return (((int64_t)side * c.pages + page) * c.heads + head) * c.page * (2 * (D / 32) * 2);
}

// The page of a position, -1 if there is none: outside the table, or its entry is no page.
__device__ __forceinline__ int page_of(const Cache& c, const int* table, int64_t width, int64_t index) {
  if (index < 0 || index >= width) return -1;
  const int page = table[index];
  return page >= 0 && page < c.pages ? page : -1;
}

struct StoreArgs {
  Cache cache;
  Heads k, v;
  const int* table;
  const int* starts;
  const int* counts;
  int64_t width;
  int batch, tokens;
};

// ---------------------------------------------------------------------------
// Append: one lane a group of 32 numbers. The lanes of a vector exchange their
// parts of its words, so that each writes 16 bytes of codes.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(const StoreArgs a) {
  constexpr int NG = D / 32, NW = D / 8;  // lanes and 32-bit words a vector
  const uint32_t id = blockIdx.x * (kThreads / NG) + threadIdx.x / NG;
  const int g = threadIdx.x % NG;
  const uint32_t T_ = a.tokens, H = a.cache.heads;
  const int t = id % T_;
  const uint32_t rest = id / T_;
  const int head = rest % H, side = (rest / H) & 1, b = rest / H / 2;
  if (b >= a.batch) return;  // the lanes of a vector leave together
  if (t >= min(a.counts[b], a.tokens)) return;
  const int64_t pos = (int64_t)a.starts[b] + t;
  const int page = pos < 0 ? -1 : page_of(a.cache, a.table + b * a.width, a.width, pos / a.cache.page);
  if (page < 0) return;
  const int slot = (int)(pos % a.cache.page);

  float x[32];
  const uint8_t* from = (side ? a.v : a.k).at(b, head, t) + 64 * g;
#pragma unroll
  for (int i = 0; i < 4; ++i) VecTraits<T>::unpack(ld16(from + 16 * i), x + 8 * i);
  float low = x[0], high = x[0];
#pragma unroll
  for (int i = 1; i < 32; ++i) {
    low = fminf(low, x[i]);
    high = fmaxf(high, x[i]);
  }
  const float s = round_to<T>((high - low) / 15.f);
  // (x - low) / s correctly rounded where it decides (ties of the rounding are exact quotients): one correction
  // of the product with the reciprocal, a plain division where that leaves the normal numbers
  uint32_t c[32];
  if (s > 1e-30f && s < 1e30f) {
    const float r = __builtin_amdgcn_rcpf(s);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float d = x[i] - low, y = d * r;
      const float f = __builtin_fmaf(__builtin_fmaf(-y, s, d), r, y);
      c[i] = (uint32_t)fminf(fmaxf(rintf(f), 0.f), 15.f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) c[i] = s > 0.f ? (uint32_t)fminf(fmaxf(rintf((x[i] - low) / s), 0.f), 15.f) : 0u;
  }

  uint32_t w[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    if constexpr (D == 128) {
      w[i] = (c[i] | (c[i + 16] << 16)) << (4 * g);
    } else {
      w[i] = (c[2 * i] | (c[2 * i + 16] << 4) | (c[2 * i + 1] << 16) | (c[2 * i + 17] << 20)) << (8 * g);
    }
  }
  // each step gives half of the words to the partner lane and takes its part of the other half
  if constexpr (NG == 4) {
    const bool up = g & 2;
#pragma unroll
    for (int i = 0; i < NW / 2; ++i) {
      const uint32_t give = up ? w[i] : w[i + NW / 2], keep = up ? w[i + NW / 2] : w[i];
      w[i] = keep | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, 0x4E, 0xF, 0xF, false);
    }
  }
  {
    const bool up = g & 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t give = up ? w[i] : w[i + 4], keep = up ? w[i + 4] : w[i];
      w[i] = keep | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, 0xB1, 0xF, 0xF, false);
    }
  }
  st16(a.cache.codes + codes_at<D>(a.cache, side, page, head) + (int64_t)slot * (D / 2) + 16 * g,
       make_uint4(w[0], w[1], w[2], w[3]));
  uint16_t* p = (uint16_t*)(a.cache.params + params_at<D>(a.cache, side, page, head)) + slot;
  p[g * a.cache.page] = (uint16_t)pack2<T>(s, 0.f);
  p[(NG + g) * a.cache.page] = (uint16_t)pack2<T>(low, 0.f);
}

// ---------------------------------------------------------------------------
// Read: D / 8 lanes a vector, 8 numbers each: one shift of 8 words.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(const StoreArgs a) {
  constexpr int NG = D / 32, L = D / 8;
  const uint32_t id = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int j = threadIdx.x % L;
  const uint32_t T_ = a.tokens, H = a.cache.heads;
  const int t = id % T_;
  const uint32_t rest = id / T_;
  const int head = rest % H, side = (rest / H) & 1, b = rest / H / 2;
  if (b >= a.batch) return;
  int page = -1;
  int64_t pos = 0;
  if (t < a.counts[b]) {
    pos = (int64_t)a.starts[b] + t;
    if (pos >= 0) page = page_of(a.cache, a.table + b * a.width, a.width, pos / a.cache.page);
  }
  uint4 y = make_uint4(0, 0, 0, 0);
  if (page >= 0) {
    const int slot = (int)(pos % a.cache.page), i = j / 2, g = i / 2;
    const uint8_t* codes = a.cache.codes + codes_at<D>(a.cache, side, page, head) + (int64_t)slot * (D / 2);
    const uint16_t* p = (const uint16_t*)(a.cache.params + params_at<D>(a.cache, side, page, head)) + slot;
    const float s = unpack1<T>(p[g * a.cache.page]), m = unpack1<T>(p[(NG + g) * a.cache.page]);
    float x[8];
    if constexpr (D == 128) {
      const uint4 u = ld16(codes + 32 * (j & 1)), v = ld16(codes + 32 * (j & 1) + 16);
      const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
      const int shift = 4 * (i / 2 + 4 * (i % 2));
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf((float)((w[e] >> shift) & 15u), s, m);
    } else {
      const uint4 u = ld16(codes + 16 * (j & 1));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = __builtin_fmaf((float)((w[e / 2] >> (4 * i + 16 * (e % 2))) & 15u), s, m);
    }
    y = VecTraits<T>::pack(x);
  }
  st16((side ? a.v : a.k).at(b, head, t) + 16 * j, y);
}

// ---------------------------------------------------------------------------
// Attention over the cache
// ---------------------------------------------------------------------------
constexpr int kTok = 32;   // tokens of a tile: one wave's step
constexpr int kRows = 16;  // query rows of a workgroup: the heads that share a key head, times the queries

struct AttendArgs {
  Cache cache;
  Heads q, o;
  const int* table;
  const int* lengths;
  float* part;   // [batch, q_heads, queries, splits, D + 2]: numbers, largest logit, sum
  int64_t width;
  int batch, q_heads, queries;
  int window, sinks;  // window 0: none
  int per, splits;    // tiles of a workgroup; workgroups of a row block
  int shift;          // log2 of the page, -1 if it is no power of two
  float scale;
};

// The tiles a sequence's queries see: [0, sink) hold the sinks, then those from the first query's window on.
struct CacheTiles {
  int n, sink, near, count;
  __device__ __forceinline__ CacheTiles(const AttendArgs& a, int b) {
    const int64_t room = a.width * a.cache.page;
    n = (int)min((int64_t)max(a.lengths[b], 0), room);
    const int lo = a.window ? max(0, n - a.queries - a.window + 1) / kTok : 0;
    sink = min((min(a.sinks, n) + kTok - 1) / kTok, lo);
    near = lo - sink;
    count = n == 0 ? 0 : sink + (n - 1) / kTok + 1 - lo;
  }
  __device__ __forceinline__ int tile(int i) const { return i < sink ? i : i + near; }
};

// Codes at bits 4 k of both halves of x as f16 numbers c 2^-24 (k even) or c 2^-20 (k odd): subnormal numbers,
// whose fraction they are. The matrix instructions take them exactly, so there is no conversion and no offset to
// take off again.
__device__ __forceinline__ uint32_t code_pair(uint32_t x, int k) {
  return (k & 2 ? x >> 8 : x) & (k & 1 ? 0x00f000f0u : 0x000f000fu);
}
constexpr float kEven = 16777216.f, kOdd = 1048576.f;  // 2^24, 2^20

// x to a packed pair of T (f) and what is left of it (r)
template <typename T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t* f, uint32_t* r) {
  *f = pack2<T>(x, y);
  *r = pack2<T>(x - unpack1<T>(*f & 0xffffu), y - unpack1<T>(*f >> 16));
}

// One tile as it is loaded.
template <int D>
struct RawTile {
  uint32_t k[2][D / 32];  // words of the lane's token
  uint32_t v[8];          // word l of 8 tokens (D = 64: 16 bits)
  u32x2_t p[2];           // 4 tokens of one row of params, K and V
};

// S = q K^T over codes: with q K = sum_g s_g (q c)_g + m_g (sum q)_g the codes go into the matrix instructions as they
// are, and the steps and minima touch 16 x 16 results instead of 16 x D numbers. O = P V the same way round: the weights
// take the values' steps, sum_t (p_t s_tg) c_t + sum_t p_t m_tg. A wave takes tiles of 32 tokens in turn, with its own
// running maximum and sums; waves and workgroups are joined at the end.
//
// q is scaled to below 2^14 by a power of two per row, exactly but for numbers 2^-28 of the row's largest. The weights with
// steps are f16, kept near 1 by the exponent `lift` of the largest step in the reference the exponentials are taken from
// (relative rounding 2^-12 against the 2^-9 of a bf16 result; f16 results add the product with what the rounding left).
// The weights of the minima are two 16-bit numbers of the cache's type: minimum and step often
// cancel in a value, so one rounding of each would count several times.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 3) void kv4_attend_kernel(const AttendArgs a) {
  constexpr int NG = D / 32, NB = D / 16;
  constexpr int kPad = D + 4;
  constexpr bool kTwo = __is_same(T, f16_t);
  __shared__ __align__(16) float merge[4][kRows][kPad];
  __shared__ float stats[4][2][kRows];
  __shared__ __align__(16) uint16_t params[4][2][2 * NG][kTok];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = lane & 15, quad = lane >> 4;
  const int kv_heads = a.cache.heads, G = a.q_heads / kv_heads, R = G * a.queries;
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int kv = id % kv_heads;
  id /= kv_heads;
  const int b = id % a.batch, r0 = id / a.batch * kRows;
  const CacheTiles tiles(a, b);
  const int first = split * a.per, last = min(first + a.per, tiles.count);
  if (first >= last && split > 0) return;  // the join does not read it

  const int r = r0 + l;  // the lane's row: head kv G + r / queries, query r % queries
  const int Q = a.queries, n = tiles.n;
  const int pos = r < R ? n - Q + r % Q : -1;
  const int p0 = n - Q, p1 = n - 1;
  const int W = a.window ? a.window : 0x7fffffff, S = a.sinks;

  const int* table = a.table + b * a.width;
  const int last_entry = (int)a.width - 1;
  // table entries of a tile's two halves (those past the table belong to tokens past the length)
  const auto entries = [&](int t, int (&entry)[2]) {
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      const int at = kTok * t + 16 * hb, i = a.shift >= 0 ? at >> a.shift : at / a.cache.page;
      entry[hb] = table[min(i, last_entry)];
    }
  };
  const auto load = [&](int t, const int (&entry)[2], RawTile<D>& x, bool (&there)[2]) {
    int page[2], slots[2];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      const int e = __builtin_amdgcn_readfirstlane(entry[hb]);
      const int at = kTok * t + 16 * hb;
      there[hb] = e >= 0 && e < a.cache.pages;
      page[hb] = there[hb] ? e : 0;
      slots[hb] = a.shift >= 0 ? at & (a.cache.page - 1) : at % a.cache.page;
      const uint8_t* kc = a.cache.codes + codes_at<D>(a.cache, 0, page[hb], kv) + slots[hb] * (D / 2);
      const uint8_t* vc = a.cache.codes + codes_at<D>(a.cache, 1, page[hb], kv) + slots[hb] * (D / 2);
      if constexpr (D == 128) {
        const frag_t y = *(const frag_t*)(kc + (uint32_t)(l * 64 + quad * 16));
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x.k[hb][e2] = y[e2];
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x.v[4 * hb + e2] = *(const uint32_t*)(vc + (uint32_t)(quad * 256 + l * 4) + 64 * e2);
      } else {
        const u32x2_t y = *(const u32x2_t*)(kc + (uint32_t)(l * 32 + quad * 8));
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) x.k[hb][e2] = y[e2];
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x.v[4 * hb + e2] = *(const uint16_t*)(vc + (uint32_t)(quad * 128 + l * 2) + 32 * e2);
      }
    }
    // lane: row lane / 8 of the params, tokens 4 (lane % 8) ..
    const int row = min(lane >> 3, 2 * NG - 1), tok = 4 * (lane & 7), hb = tok >> 4;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int64_t b0 = params_at<D>(a.cache, side, page[0], kv) + 2 * slots[0];
      const int64_t b1 = params_at<D>(a.cache, side, page[1], kv) + 2 * slots[1];
      x.p[side] = *(const u32x2_t*)(a.cache.params + (hb ? b1 : b0) + 2 * (row * a.cache.page + (tok & 15)));
    }
  };

  // the first tiles are on their way while q is prepared
  RawTile<D> x;
  bool there[2] = {};
  int entry[2] = {};
  if (first + wave < last) {
    entries(tiles.tile(first + wave), entry);
    load(tiles.tile(first + wave), entry, x, there);
    entries(tiles.tile(min(first + wave + 4, last - 1)), entry);
  }

  // q as B operand, f16 numbers in the codes' order, and its sums over the groups in three parts of T
  frag_t q[NG];
  frag_t qsum = {0, 0, 0, 0};
  float c;
  {
    const uint8_t* row = (const uint8_t*)a.q.at(b, kv * G + min(r, R - 1) / Q, min(r, R - 1) % Q) + 8 * quad;
    float f[NG][8];  // [k][e]: number 16 k + 4 quad + e, k = 2 g + e / 4
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x2_t y = *(const u32x2_t*)(row + 32 * (2 * g + u));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[g][4 * u + e] = r < R ? unpack1<T>(e & 1 ? y[e / 2] >> 16 : y[e / 2] & 0xffffu) : 0.f;
          top = fmaxf(top, fabsf(f[g][4 * u + e]));
        }
      }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const int e2 = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
    c = ldexpf(a.scale * 1.44269504f, e2 + 10);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sum = 0.f, z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum += f[g][e];
        // codes at odd places are 16 times as large
        z[e] = ldexpf(f[g][e], 14 - e2 - (D == 128 ? 4 * (g & 1) : 4 * (e / 4)));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        q[g][e] = D == 128 ? pack2<f16_t>(z[e], z[4 + e]) : pack2<f16_t>(z[2 * e], z[2 * e + 1]);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      sum = ldexpf(sum, -10 - e2);
      const float s0 = round_to<T>(sum), s1 = round_to<T>(sum - s0), s2 = sum - s0 - s1;
      if (quad == g) qsum = (frag_t){pack2<T>(s0, s1), pack2<T>(s2, 0.f), 0, 0};
    }
  }

  f32x4_t o[NB] = {}, mins = {};
  float m = -INFINITY, ref = 0.f, sum = 0.f;
  uint32_t most = 0;  // the largest step so far, as its bits
  int lift = 0;       // its exponent
  for (int it = first + wave; it < last; it += 4) {
    const int j0 = tiles.tile(it) * kTok;
    RawTile<D> now = x;
    const bool there0 = there[0], there1 = there[1];
    if (it + 4 < last) {
      load(tiles.tile(it + 4), entry, x, there);
      entries(tiles.tile(min(it + 8, last - 1)), entry);
    }
    const bool all = there0 && there1 && p0 >= 0 && j0 + kTok - 1 <= p0 && (p1 - j0 < W || j0 + kTok - 1 < S);
    if (!all) {  // what the params hold for tokens that no row sees is not used
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + 4 * (lane & 7) + e;
        const bool some = ((lane & 7) < 4 ? there0 : there1) && j <= p1 && (p0 - j < W || j < S);
        const uint32_t keep = some ? 0xffffffffu : e & 1 ? 0xffffu : 0xffff0000u;
        now.p[0][e / 2] &= keep;
        now.p[1][e / 2] &= keep;
      }
    }

    // the tile's params by way of LDS: every lane needs 4 tokens of every row
    uint16_t(*par)[2 * NG][kTok] = params[wave];
    if (NG == 4 || lane < 32) {
      *(u32x2_t*)&par[0][lane >> 3][4 * (lane & 7)] = now.p[0];
      *(u32x2_t*)&par[1][lane >> 3][4 * (lane & 7)] = now.p[1];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();

    // logits of tokens 16 hb + 4 quad + i for row l, in units of 1 / c
    float s[8];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      const uint32_t low = par[0][NG + quad % NG][16 * hb + l];
      const uint32_t pair = quad < NG ? low | (low << 16) : 0;
      f32x4_t y = mfma16<T>((frag_t){pair, pair, 0, 0}, qsum, (f32x4_t){0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        frag_t f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f[e] = D == 128 ? code_pair(now.k[hb][e], g) : code_pair(now.k[hb][e & 1], 2 * g + e / 2);
        const f32x4_t acc = mfma16<f16_t>(f, q[g], (f32x4_t){0.f, 0.f, 0.f, 0.f});
        const u32x2_t ps = *(const u32x2_t*)&par[0][g][16 * hb + 4 * quad];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = __builtin_fmaf(unpack1<T>(i & 1 ? ps[i / 2] >> 16 : ps[i / 2] & 0xffffu), acc[i], y[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * hb + i] = y[i];
    }
    if (!all) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + 16 * (i >> 2) + 4 * quad + (i & 3);
        const bool see = (i < 4 ? there0 : there1) && j <= pos && (pos - j < W || j < S);
        s[i] = see ? s[i] : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(fmaxf(top, __shfl_xor(top, 32)), m);
    // steps are not negative, so their bits order them
    const uint32_t b0 = now.p[1][0], b1 = now.p[1][1];
    const uint32_t steps = lane < 8 * NG ? max(max(b0 & 0xffffu, b0 >> 16), max(b1 & 0xffffu, b1 >> 16)) : 0u;
    // a new reference where a row's largest logit has grown by more than 4 in log2, or the largest step by a power of two:
    // until then weights stay below 2^5
    if (__any((top - m) * c > 4.f || (m == -INFINITY && top > m) || steps > (most | (kTwo ? 0x3ffu : 0x7fu)))) {
      uint32_t big = steps;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) big = max(big, (uint32_t)__shfl_xor((int)big, d));
      most = max(most, big);
      const int lifted = kTwo ? (int)(most >> 10) - 14 : min(max((int)(most >> 7) - 126, -100), 100);
      const float next = (top == -INFINITY ? 0.f : top * c) + (float)lifted;
      const float f = m == -INFINITY ? 0.f : exp2_raw(ref - next);
      sum *= f;
#pragma unroll
      for (int i = 0; i < NB; ++i) o[i] *= f;
      mins *= kTwo ? ldexpf(f, lifted - lift) : f;
      m = top;
      ref = next;
      lift = lifted;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = exp2_raw(__builtin_fmaf(s[i], c, -ref));
      sum += s[i];
    }

    // sum_t p_t m_t: rows g of the A operand, in the tokens' order of s
    {
      const u32x2_t m0 = *(const u32x2_t*)&par[1][NG + l % NG][4 * quad];
      const u32x2_t m1 = *(const u32x2_t*)&par[1][NG + l % NG][16 + 4 * quad];
      const frag_t fm = {m0[0], m0[1], m1[0], m1[1]};
      frag_t fp, fr;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t hi, lo;
        // f16: without the steps' exponent, which may put weights past its range
        if constexpr (kTwo) {
          split_pair<T>(ldexpf(s[2 * e], lift), ldexpf(s[2 * e + 1], lift), &hi, &lo);
        } else {
          split_pair<T>(s[2 * e], s[2 * e + 1], &hi, &lo);
        }
        fp[e] = hi, fr[e] = lo;
      }
      mins = mfma16<T>(fm, fp, mins);
      mins = mfma16<T>(fm, fr, mins);
    }
    // sum_t p_t s_t c_t
    uint32_t lo[4], hi[4];
    if constexpr (D == 128) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = __builtin_amdgcn_perm(now.v[2 * e + 1], now.v[2 * e], 0x05040100u);
        hi[e] = __builtin_amdgcn_perm(now.v[2 * e + 1], now.v[2 * e], 0x07060302u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) lo[e] = now.v[2 * e] | (now.v[2 * e + 1] << 16);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float w[8];
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        const u32x2_t ps = *(const u32x2_t*)&par[1][g][16 * hb + 4 * quad];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[4 * hb + i] = s[4 * hb + i] * unpack1<T>(i & 1 ? ps[i / 2] >> 16 : ps[i / 2] & 0xffffu);
      }
      frag_t fw, fr;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kTwo) {
          uint32_t h2, l2;
          split_pair<f16_t>(w[2 * e], w[2 * e + 1], &h2, &l2);
          fw[e] = h2, fr[e] = l2;
        } else {
          fw[e] = pack2<f16_t>(w[2 * e], w[2 * e + 1]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        frag_t f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = D == 128 ? code_pair(u ? hi[e] : lo[e], g) : code_pair(lo[e], 2 * g + u);
        o[2 * g + u] = mfma16<f16_t>(f, fw, o[2 * g + u]);
        if constexpr (kTwo) o[2 * g + u] = mfma16<f16_t>(f, fr, o[2 * g + u]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // the waves' sums, joined by way of LDS
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const float add = kTwo ? ldexpf(mins[i / 2], -lift) : mins[i / 2], unit = (D == 128 ? i / 2 : i) & 1 ? kOdd : kEven;
    f32x4_t y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(o[i][e], unit, add);
    *(f32x4_t*)&merge[wave][l][16 * i + 4 * quad] = y;
  }
  if (quad == 0) {
    stats[wave][0][l] = ref;
    stats[wave][1][l] = sum;
  }
  __syncthreads();
  const int row = tid / 16, d0 = tid % 16 * (D / 16);
  if (r0 + row >= R) return;
  // waves without a visible token have sum 0 and a reference that is no maximum: they are left out
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = stats[w][1][row] != 0.f ? fmaxf(top, stats[w][0][row]) : top;
  const float base = top == -INFINITY ? 0.f : top;
  float y[D / 16] = {}, total = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = stats[w][1][row] != 0.f ? exp2_raw(stats[w][0][row] - base) : 0.f;
    total = __builtin_fmaf(f, stats[w][1][row], total);
#pragma unroll
    for (int e = 0; e < D / 16; ++e) y[e] = __builtin_fmaf(f, merge[w][row][d0 + e], y[e]);
  }
  const int head = kv * G + (r0 + row) / Q, query = (r0 + row) % Q;
  if (a.splits == 1) {
    const float f = total != 0.f ? 1.f / total : 0.f;
    uint32_t z[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) z[e] = pack2<T>(y[2 * e] * f, y[2 * e + 1] * f);
    uint32_t* to = (uint32_t*)(a.o.at(b, head, query) + 2 * d0);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) to[e] = total != 0.f ? z[e] : 0u;
  } else {
    float* to = a.part + (((int64_t)(b * a.q_heads + head) * Q + query) * a.splits + split) * (D + 2);
#pragma unroll
    for (int e = 0; e < D / 16; ++e) to[d0 + e] = y[e];
    if (d0 == 0) {
      to[D] = top;
      to[D + 1] = total;
    }
  }
}

// Joins the parts of one row: 16 groups of 16 lanes take parts in turn.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void kv4_join_kernel(const AttendArgs a) {
  __shared__ float numbers[16][D + 4];
  __shared__ float stats[2][16];
  const int Q = a.queries, query = blockIdx.x % Q, bh = blockIdx.x / Q;
  const int b = bh / a.q_heads, head = bh % a.q_heads;
  const CacheTiles tiles(a, b);
  const int parts = max(1, (tiles.count + a.per - 1) / a.per);
  const int g = threadIdx.x / 16, d0 = threadIdx.x % 16 * (D / 16);
  const float* from = a.part + (int64_t)blockIdx.x * a.splits * (D + 2);
  float top = -INFINITY;
  for (int i = g; i < parts; i += 16) top = fmaxf(top, from[(int64_t)i * (D + 2) + D]);
  float base = top == -INFINITY ? 0.f : top;
  float y[D / 16] = {}, total = 0.f;
  for (int i = g; i < parts; i += 16) {
    const float* p = from + (int64_t)i * (D + 2);
    const float f = exp2_raw(p[D] - base);
    total = __builtin_fmaf(f, p[D + 1], total);
#pragma unroll
    for (int e = 0; e < D / 16; ++e) y[e] = __builtin_fmaf(f, p[d0 + e], y[e]);
  }
#pragma unroll
  for (int e = 0; e < D / 16; ++e) numbers[g][d0 + e] = y[e];
  if (d0 == 0) {
    stats[0][g] = top;
    stats[1][g] = total;
  }
  __syncthreads();
  if ((int)threadIdx.x >= D / 2) return;
  top = stats[0][0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, stats[0][i]);
  base = top == -INFINITY ? 0.f : top;
  total = 0.f;
  float y0 = 0.f, y1 = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float f = exp2_raw(stats[0][i] - base);
    total = __builtin_fmaf(f, stats[1][i], total);
    y0 = __builtin_fmaf(f, numbers[i][2 * threadIdx.x], y0);
    y1 = __builtin_fmaf(f, numbers[i][2 * threadIdx.x + 1], y1);
  }
  const float f = total != 0.f ? 1.f / total : 0.f;
  ((uint32_t*)a.o.at(b, head, query))[threadIdx.x] = total != 0.f ? pack2<T>(y0 * f, y1 * f) : 0u;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_cache(const char* what, Cache* c, void* codes, void* params, int64_t pages, int64_t heads, int64_t page,
                int64_t dim, int dtype) {
  PKM_REQUIRE(pages >= 0 && heads > 0 && page > 0, PKM_ERR_INVALID_ARGUMENT, "%s: bad cache sizes", what);
  PKM_REQUIRE((dim == 64 || dim == 128) && (dtype == PKM_DTYPE_BF16 || dtype == PKM_DTYPE_F16), PKM_ERR_UNSUPPORTED,
              "%s: head dims 64 and 128 in bf16 and f16 are supported", what);
  PKM_REQUIRE(page % 16 == 0 && page <= 4096, PKM_ERR_UNSUPPORTED,
              "%s: pages of a multiple of 16 tokens, 4096 at most, are supported", what);
  PKM_REQUIRE(pages < (1ll << 31) && heads < (1 << 20), PKM_ERR_UNSUPPORTED, "%s: too many pages or heads", what);
  PKM_REQUIRE(codes != nullptr && params != nullptr && (((uintptr_t)codes | (uintptr_t)params) & 15) == 0,
              PKM_ERR_INVALID_ARGUMENT, "%s: codes and params have to be given, 16-byte aligned", what);
  *c = {(uint8_t*)codes, (uint8_t*)params, pages, (int)heads, (int)page};
  return PKM_OK;
}

int check_rows(const char* what, const char* name, const pkm_heads_t* x) {
  PKM_REQUIRE(x != nullptr && x->data != nullptr, PKM_ERR_INVALID_ARGUMENT, "%s: %s is NULL", what, name);
  PKM_REQUIRE(((uintptr_t)x->data & 15) == 0 && x->batch % 8 == 0 && x->head % 8 == 0 && x->token % 8 == 0 &&
                  x->batch >= 0 && x->head >= 0 && x->token >= 0,
              PKM_ERR_UNSUPPORTED, "%s: %s needs 16-byte aligned data and strides >= 0 that are multiples of 8", what,
              name);
  return PKM_OK;
}

Heads heads(const pkm_heads_t* x) { return {(uint8_t*)x->data, x->batch, x->head, x->token}; }

int store_args(const char* what, StoreArgs* a, int64_t dim, int dtype, const pkm_heads_t* k, const pkm_heads_t* v,
               const int32_t* table, int64_t width, const int32_t* starts, const int32_t* counts, int64_t batch,
               int64_t tokens) {
  int rc;
  if ((rc = check_rows(what, "k", k)) || (rc = check_rows(what, "v", v))) return rc;
  PKM_REQUIRE(starts != nullptr && counts != nullptr && (table != nullptr || width == 0), PKM_ERR_INVALID_ARGUMENT,
              "%s: table, starts and counts have to be given", what);
  PKM_REQUIRE(batch < (1ll << 31) && tokens < (1ll << 31) && 2 * batch * tokens < (1ll << 31) / a->cache.heads,
              PKM_ERR_UNSUPPORTED, "%s: too many tokens", what);
  a->k = heads(k), a->v = heads(v);
  a->table = table, a->starts = starts, a->counts = counts, a->width = width;
  a->batch = (int)batch, a->tokens = (int)tokens;
  (void)dim, (void)dtype;
  return PKM_OK;
}

template <bool APPEND, typename T, int D>
void launch_store(const StoreArgs& a, hipStream_t st) {
  const int64_t vectors = 2ll * a.batch * a.tokens * a.cache.heads;
  constexpr int per = kThreads / (APPEND ? D / 32 : D / 8);
  const unsigned grid = (unsigned)((vectors + per - 1) / per);
  if constexpr (APPEND) {
    kv4_append_kernel<T, D><<<grid, kThreads, 0, st>>>(a);
  } else {
    kv4_read_kernel<T, D><<<grid, kThreads, 0, st>>>(a);
  }
}

template <bool APPEND>
int run_store(const char* what, const StoreArgs& a, int64_t dim, int dtype, void* stream) {
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKM_DTYPE_BF16) {
    dim == 128 ? launch_store<APPEND, bf16_t, 128>(a, st) : launch_store<APPEND, bf16_t, 64>(a, st);
  } else {
    dim == 128 ? launch_store<APPEND, f16_t, 128>(a, st) : launch_store<APPEND, f16_t, 64>(a, st);
  }
  return pkm_check_launch(what);
}

// Tiles of a workgroup and workgroups of a row block, from sizes alone: enough workgroups to fill the card
// a few times over, tiles enough for 4 waves each.
void split_plan(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t queries, int64_t width, int64_t page,
                int64_t window, int64_t sinks, int* per, int* splits) {
  const int64_t rows = (q_heads / kv_heads * queries + kRows - 1) / kRows;
  int64_t most = (width * page + kTok - 1) / kTok;
  if (window > 0) {
    const int64_t seen = (window + queries) / kTok + 2 + (sinks + kTok - 1) / kTok;
    if (seen < most) most = seen;
  }
  const int64_t blocks = batch * kv_heads * rows;
  int64_t each = (most * blocks + 2047) / 2048;
  if (each < 8) each = 8;
  if (most < 1) most = 1;
  *per = (int)each;
  *splits = (int)((most + each - 1) / each);
}

int64_t part_bytes(int64_t batch, int64_t q_heads, int64_t queries, int64_t dim, int splits) {
  return splits == 1 ? 0 : batch * q_heads * queries * splits * (dim + 2) * (int64_t)sizeof(float);
}

template <typename T, int D>
void launch_attend(const AttendArgs& a, hipStream_t st) {
  const int rows = (a.q_heads / a.cache.heads * a.queries + kRows - 1) / kRows;
  kv4_attend_kernel<T, D><<<(unsigned)(a.batch * a.cache.heads * rows * a.splits), kThreads, 0, st>>>(a);
  if (a.splits > 1) kv4_join_kernel<T, D><<<(unsigned)(a.batch * a.q_heads * a.queries), kThreads, 0, st>>>(a);
}

}  // namespace
}  // namespace pkm

using namespace pkm;

extern "C" int pkm_kv4_append(void* codes, void* params, int64_t pages, int64_t kv_heads, int64_t page, int64_t dim,
                              int dtype, const pkm_heads_t* k, const pkm_heads_t* v, const int32_t* table,
                              int64_t width, const int32_t* starts, const int32_t* counts, int64_t batch,
                              int64_t tokens, void* stream) {
  const char* what = "pkm_kv4_append";
  PKM_REQUIRE(batch >= 0 && tokens >= 0 && width >= 0, PKM_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (batch == 0 || tokens == 0 || pages == 0) return PKM_OK;
  StoreArgs a = {};
  int rc = check_cache(what, &a.cache, codes, params, pages, kv_heads, page, dim, dtype);
  if (rc != PKM_OK) return rc;
  if ((rc = store_args(what, &a, dim, dtype, k, v, table, width, starts, counts, batch, tokens))) return rc;
  return run_store<true>(what, a, dim, dtype, stream);
}

extern "C" int pkm_kv4_read(const void* codes, const void* params, int64_t pages, int64_t kv_heads, int64_t page,
                            int64_t dim, int dtype, const int32_t* table, int64_t width, const int32_t* starts,
                            const int32_t* counts, int64_t batch, int64_t tokens, const pkm_heads_t* k,
                            const pkm_heads_t* v, void* stream) {
  const char* what = "pkm_kv4_read";
  PKM_REQUIRE(batch >= 0 && tokens >= 0 && width >= 0, PKM_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (batch == 0 || tokens == 0) return PKM_OK;
  StoreArgs a = {};
  int rc = check_cache(what, &a.cache, const_cast<void*>(codes), const_cast<void*>(params), pages, kv_heads, page, dim,
                       dtype);
  if (rc != PKM_OK) return rc;
  if ((rc = store_args(what, &a, dim, dtype, k, v, table, width, starts, counts, batch, tokens))) return rc;
  return run_store<false>(what, a, dim, dtype, stream);
}

extern "C" size_t pkm_kv4_attend_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t queries,
                                                int64_t dim, int64_t width, int64_t page, int64_t window,
                                                int64_t sinks) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || queries <= 0 || dim <= 0 || width < 0 || page <= 0) return 0;
  int per, splits;
  split_plan(batch, q_heads, kv_heads, queries, width, page, window, sinks, &per, &splits);
  return (size_t)part_bytes(batch, q_heads, queries, dim, splits);
}

extern "C" int pkm_kv4_attend(const void* codes, const void* params, int64_t pages, int64_t kv_heads, int64_t page,
                              int64_t dim, int dtype, const pkm_heads_t* q, const int32_t* table, int64_t width,
                              const int32_t* lengths, int64_t batch, int64_t q_heads, int64_t queries, int64_t window,
                              int64_t sinks, float scale, const pkm_heads_t* out, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* what = "pkm_kv4_attend";
  PKM_REQUIRE(batch >= 0 && queries >= 0 && width >= 0 && q_heads > 0 && kv_heads > 0 && window >= 0 && sinks >= 0,
              PKM_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  PKM_REQUIRE(q_heads % kv_heads == 0, PKM_ERR_INVALID_ARGUMENT, "%s: %lld query heads do not share %lld key heads",
              what, (long long)q_heads, (long long)kv_heads);
  PKM_REQUIRE(scale > 0.f && scale <= 3.0e38f, PKM_ERR_INVALID_ARGUMENT, "%s: scale has to be positive and finite", what);
  if (batch == 0 || queries == 0) return PKM_OK;
  AttendArgs a = {};
  int rc = check_cache(what, &a.cache, const_cast<void*>(codes), const_cast<void*>(params), pages, kv_heads, page, dim,
                       dtype);
  if (rc != PKM_OK) return rc;
  if ((rc = check_rows(what, "q", q)) || (rc = check_rows(what, "out", out))) return rc;
  PKM_REQUIRE(pages > 0, PKM_ERR_UNSUPPORTED, "%s: the cache has no pages", what);
  PKM_REQUIRE(lengths != nullptr && (table != nullptr || width == 0), PKM_ERR_INVALID_ARGUMENT,
              "%s: table and lengths have to be given", what);
  PKM_REQUIRE(width < (1ll << 31) / page && batch < (1 << 24) && q_heads < (1 << 20) && queries < (1 << 20) &&
                  batch * q_heads * queries < (1ll << 24),
              PKM_ERR_UNSUPPORTED, "%s: too many tokens or rows", what);
  split_plan(batch, q_heads, kv_heads, queries, width, page, window, sinks, &a.per, &a.splits);
  PKM_REQUIRE(workspace_bytes >= (size_t)part_bytes(batch, q_heads, queries, dim, a.splits) &&
                  (a.splits == 1 || workspace != nullptr),
              PKM_ERR_WORKSPACE, "%s: workspace too small", what);
  a.q = heads(q), a.o = heads(out);
  a.table = table, a.lengths = lengths, a.part = (float*)workspace, a.width = width;
  a.batch = (int)batch, a.q_heads = (int)q_heads, a.queries = (int)queries;
  const int64_t far = 1 << 30;
  a.window = (int)(window < far ? window : 0), a.sinks = (int)(sinks < far ? sinks : far);
  a.scale = scale;
  a.shift = (page & (page - 1)) == 0 ? __builtin_ctzll((unsigned long long)page) : -1;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKM_DTYPE_BF16) {
    dim == 128 ? launch_attend<bf16_t, 128>(a, st) : launch_attend<bf16_t, 64>(a, st);
  } else {
    dim == 128 ? launch_attend<f16_t, 128>(a, st) : launch_attend<f16_t, 64>(a, st);
  }
  return pkm_check_launch(what);
}
