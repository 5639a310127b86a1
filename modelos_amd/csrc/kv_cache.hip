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
#include <algorithm>

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
  int shift;  // log2 of the page, -1 if it is no power of two
};

// Where token t of a vector's sequence lies: its page (-1: nowhere) and slot.
struct Place {
  int page, slot;
  __device__ __forceinline__ Place(const StoreArgs& a, int b, int t) {
    const int64_t pos = (int64_t)a.starts[b] + t;
    const uint32_t at = (uint32_t)pos;  // below 2^32
    const uint32_t index = a.shift >= 0 ? at >> a.shift : at / (uint32_t)a.cache.page;
    slot = (int)(at - index * (uint32_t)a.cache.page);
    page = pos < 0 ? -1 : page_of(a.cache, a.table + b * a.width, a.width, index);
  }
};

// ---------------------------------------------------------------------------
// Append: one lane a group of 32 numbers. The lanes of a vector exchange their
// parts of its words, so that each writes 16 bytes of codes. Bound by memory: 25 000
// tokens of 8 heads of 128 (134 MB) in 35 us, 3.9 TB/s.
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
  const Place place(a, b, t);
  const int page = place.page, slot = place.slot;
  if (page < 0) return;

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
// Read: D / 8 lanes a vector, 8 numbers each: one shift of 8 words. Bound by memory: the
// same tokens with the zeros behind the shorter sequences (196 MB) in 46 us, 4.2 TB/s.
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
  int page = -1, slot = 0;
  if (t < a.counts[b]) {
    const Place place(a, b, t);
    page = place.page, slot = place.slot;
  }
  uint4 y = make_uint4(0, 0, 0, 0);
  if (page >= 0) {
    const int i = j / 2, g = i / 2;
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
constexpr int kGroups = 768;  // workgroups of a large call: 3 on each of 256 CUs run at once

struct AttendArgs {
  Cache cache;
  Heads q, o;
  const int* table;
  const int* lengths;
  float* part;   // [workgroups + segments, 16 rows, D + 2]: numbers, reference, sum
  int64_t width;
  int batch, q_heads, queries;
  int window, sinks;  // window 0: none
  int rows, groups;   // row blocks of a key head; workgroups
  int cut;            // workgroups less what the segments' last pieces waste, where each is cut on its own
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

// A segment is the tiles of one sequence, key head and row block. How the workgroups share all segments is worked out on the
// device, where the lengths are:
//   whole: with many tiles a workgroup, all segments in a row, in that order, are cut into equal shares, so that
//     ragged lengths cost nothing; a share may reach over several segments. (64 sequences of 4000 to 16000 tokens, 8 key
//     heads: 180 us; cut segment by segment into pieces of one size, 186 to 215 with the size.)
//   else each segment is cut on its own, as starting a second segment costs more than the balance gains
//     (window of 1024, 64 sequences: 27 us against 34), into pieces that all run at once (32 us in two rounds).
// A workgroup's part of a segment goes to a slot of the workspace, or to the output if it is the whole segment.
struct Shares {
  bool whole;
  int per;         // tiles of a workgroup
  int64_t before;  // tiles (whole) or workgroups of the sequences before b
  int b, count;    // a sequence and its segments' tiles
  // of a segment, not whole: workgroups and their tiles
  __device__ __forceinline__ int pieces() const { return (count + per - 1) / per; }
  __device__ __forceinline__ int piece() const { return (count + pieces() - 1) / pieces(); }
};

// Sum over the lanes up to and with the own one.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp_add_u32(uint32_t x) {
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = dpp_add_u32<0x111>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add_u32<0x112>(x);
  x = dpp_add_u32<0x114>(x);
  x = dpp_add_u32<0x118>(x);
  x = dpp_add_u32<0x142, 0xa>(x);         // the rows' sums to the rows behind
  return dpp_add_u32<0x143, 0xc>(x);
}

// x / y of numbers that are not negative: in 32 bits where x has no more (a 64-bit division takes a microsecond).
__device__ __forceinline__ int64_t quotient(int64_t x, int y) {
  return (uint64_t)x >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}

// The shares, and the sequence that holds the first tile of workgroup `group` (the batch's size if there is none); or,
// with group < 0, sequence b. Each wave works them out by itself: 64 sequences at a time.
__device__ __forceinline__ Shares shares(const AttendArgs& a, int group, int b) {
  const int lane = threadIdx.x & 63;
  const int64_t heads = (int64_t)a.cache.heads * a.rows;
  const auto count = [&](int i) { return i < a.batch ? CacheTiles(a, i).count : 0; };
  // counts are below 2^25 (the entry point checks the table's width), 64 of them below 2^31
  const uint32_t mine = count(lane), sums = wave_scan(mine);
  int64_t total = (uint32_t)__builtin_amdgcn_readlane((int)sums, 63);
  for (int i = 64; i < a.batch; i += 64)
    total += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(count(i + lane)), 63);
  total *= heads;
  Shares r;
  const int64_t even = quotient(total + a.groups - 1, a.groups);
  r.whole = even >= 64;
  r.per = (int)(r.whole ? even : max(quotient(total + a.cut - 1, a.cut), (int64_t)4));
  const int64_t first = r.whole ? (int64_t)group * r.per : group;
  r.b = a.batch;
  r.before = 0;
  int64_t passed = 0;  // of the sequences before
  for (int i0 = 0; i0 < a.batch; i0 += 64) {
    uint32_t t = i0 ? (uint32_t)count(i0 + lane) : mine;
    if (!r.whole) t = (t + r.per - 1) / (uint32_t)r.per;
    const uint32_t upto = i0 || !r.whole ? wave_scan(t) : sums;
    const int64_t scan = passed + upto * heads, own = t * heads;
    const uint64_t here = __ballot(group < 0 ? i0 + lane == b : t > 0 && scan - own <= first && first < scan);
    if (here) {
      const int at = __builtin_ctzll(here);
      r.b = i0 + at;
      r.before = passed + (uint32_t)__builtin_amdgcn_readlane((int)(upto - t), at) * heads;
      break;
    }
    passed += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63) * heads;
  }
  r.b = __builtin_amdgcn_readfirstlane(r.b);
  r.count = r.b < a.batch ? CacheTiles(a, r.b).count : 0;
  return r;
}

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
// running maximum and sums; waves and workgroups are joined at the end. The next tile is on its way while one is
// worked on, at three workgroups a CU.
//
// Bound by memory where there are many tiles: 64 sequences of 4000 to 16000 tokens, 32 / 8 heads of 128 (828 MB) in
// 176 to 182 us, 4.5 to 4.7 TB/s of the 4.7 that a large copy reaches; one of 131072 tokens (168 MB) in
// 40 us, of which 6 are its start and end. 415 vector instructions a tile keep the vector units busy 63 % of the cycles. (Codes widened to 16 + c in the query's type, with
// products that take the 16 off again, 349 us for the first; 128 registers for a fourth workgroup spill, 2 times slower.)
//
// q is scaled to below 2^14 by a power of two per row, exactly but for numbers 2^-28 of the row's largest. The weights with
// steps are f16, kept near 1 by 2^-lift, which brings the wave's largest step so far to between 1/2 and 1
// (rounding 2^-11 of a product against the 2^-8 of a bf16 result, and 2^-25 below 2^-14: products 2^-14 of the
// largest lose bits; f16 results add the product with what the rounding left). The weights of the minima
// are two 16-bit numbers of the cache's type: minimum and step often cancel in a value, so one rounding of each would
// count several times. They do without 2^-lift: minima may be large where all steps are 0.
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
  const int group = blockIdx.x;
  const Shares share = shares(a, group, 0);
  const int heads = kv_heads * a.rows;
  int b = share.b;
  if (b >= a.batch) return;
  int64_t before = share.before, at, end;  // tiles before the sequence's; the next tile and the share's end
  int part_head;                           // key head and row block of the segment
  if (share.whole) {
    at = (int64_t)group * share.per;
    end = at + share.per;
    part_head = (int)quotient(at - before, share.count);
  } else {
    const uint32_t piece = (uint32_t)(group - before), pieces = share.pieces();
    part_head = (int)(piece / pieces);
    before = 0;
    at = (int64_t)part_head * share.count + piece % pieces * share.piece();
    end = min(at + share.piece(), (int64_t)(part_head + 1) * share.count);
    if (at >= end) return;  // the join does not read it
  }
  for (;;) {
  const CacheTiles tiles(a, b);
  const int64_t start = before + (int64_t)part_head * tiles.count;
  const int first = (int)(at - start), last = (int)min((int64_t)tiles.count, end - start);
  const int kv = part_head / a.rows, r0 = part_head % a.rows * kRows;

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
  // bytes of a page's codes over all heads; the params of the same tokens take a quarter
  const int64_t page_bytes = (int64_t)a.cache.heads * a.cache.page * (D / 2);
  const uint8_t* const kcodes = a.cache.codes + (int64_t)kv * a.cache.page * (D / 2);
  const uint8_t* const vcodes = kcodes + a.cache.pages * page_bytes;
  const uint8_t* const kparams = a.cache.params + (int64_t)kv * a.cache.page * (D / 8);
  const uint8_t* const vparams = kparams + a.cache.pages * page_bytes / 4;
  // a lane's params: row lane / 8, tokens 4 (lane % 8) ..
  const uint32_t param_at = 2 * (min(lane >> 3, 2 * NG - 1) * a.cache.page + 4 * (lane & 3));
  const auto load = [&](int t, const int (&entry)[2], RawTile<D>& x, bool (&there)[2]) {
    int64_t pofs[2];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      const int e = __builtin_amdgcn_readfirstlane(entry[hb]);
      const int at = kTok * t + 16 * hb;
      there[hb] = e >= 0 && e < a.cache.pages;
      const int slot = a.shift >= 0 ? at & (a.cache.page - 1) : at % a.cache.page;
      const int64_t page = (there[hb] ? e : 0) * page_bytes;
      // 16 tokens' codes each, addressed by the lane's place alone
      const __amdgpu_buffer_rsrc_t kc = row_rsrc(kcodes + (page + slot * (D / 2)), 8 * D);
      const __amdgpu_buffer_rsrc_t vc = row_rsrc(vcodes + (page + slot * (D / 2)), 8 * D);
      pofs[hb] = page / 4 + 2 * slot;
      if constexpr (D == 128) {
        const frag_t y = __builtin_amdgcn_raw_buffer_load_b128(kc, l * 64 + quad * 16, 0, 0);
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x.k[hb][e2] = y[e2];
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x.v[4 * hb + e2] = __builtin_amdgcn_raw_buffer_load_b32(vc, quad * 256 + l * 4 + 64 * e2, 0, 0);
      } else {
        const u32x2_t y = __builtin_amdgcn_raw_buffer_load_b64(kc, l * 32 + quad * 8, 0, 0);
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) x.k[hb][e2] = y[e2];
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x.v[4 * hb + e2] = __builtin_amdgcn_raw_buffer_load_b16(vc, quad * 128 + l * 2 + 32 * e2, 0, 0);
      }
    }
    const int64_t at = (lane & 4 ? pofs[1] : pofs[0]) + param_at;
    x.p[0] = *(const u32x2_t*)(kparams + at);
    x.p[1] = *(const u32x2_t*)(vparams + at);
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
  int lift = 0;       // its exponent; o is in units of 2^lift
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
    // until then weights stay below 2^4
    if (__any((top - m) * c > 4.f || (m == -INFINITY && top > m) || steps > (most | (kTwo ? 0x3ffu : 0x7fu)))) {
      uint32_t big = steps;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) big = max(big, (uint32_t)__shfl_xor((int)big, d));
      most = max(most, (uint32_t)__builtin_amdgcn_readfirstlane((int)big));
      const int lifted = kTwo ? (int)(most >> 10) - 14 : min(max((int)(most >> 7) - 126, -100), 100);
      const float next = top == -INFINITY ? 0.f : top * c;
      const float f = m == -INFINITY ? 0.f : exp2_raw(ref - next), fo = ldexpf(f, lift - lifted);
      sum *= f;
#pragma unroll
      for (int i = 0; i < NB; ++i) o[i] *= fo;
      mins *= f;
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
        split_pair<T>(s[2 * e], s[2 * e + 1], &hi, &lo);
        fp[e] = hi, fr[e] = lo;
      }
      mins = mfma16<T>(fm, fp, mins);
      mins = mfma16<T>(fm, fr, mins);
    }
    // sum_t p_t s_t c_t
    const float up = ldexpf(1.f, -lift);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= up;
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
      // f16: group by group, or the groups' pairs of operands together take 50 registers more than there are
      if constexpr (kTwo) __builtin_amdgcn_sched_barrier(0);
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
    const float unit = ldexpf((D == 128 ? i / 2 : i) & 1 ? kOdd : kEven, lift);
    f32x4_t y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(o[i][e], unit, mins[i / 2]);
    *(f32x4_t*)&merge[wave][l][16 * i + 4 * quad] = y;
  }
  if (quad == 0) {
    stats[wave][0][l] = ref;
    stats[wave][1][l] = sum;
  }
  __syncthreads();
  const int row = tid / 16, d0 = tid % 16 * (D / 16);
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
  if (r0 + row >= R) {
  } else if (first == 0 && last == tiles.count) {
    const float f = total != 0.f ? 1.f / total : 0.f;
    uint32_t z[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) z[e] = pack2<T>(y[2 * e] * f, y[2 * e + 1] * f);
    uint32_t* to = (uint32_t*)(a.o.at(b, head, query) + 2 * d0);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) to[e] = total != 0.f ? z[e] : 0u;
  } else {
    const int64_t slot = share.whole ? group + (int64_t)b * heads + part_head : group;
    float* to = a.part + slot * (kRows * (D + 2));
#pragma unroll
    for (int e = 0; e < D / 16; ++e) to[row * D + d0 + e] = y[e];
    if (d0 == 0) {
      to[kRows * D + 2 * row] = top;
      to[kRows * D + 2 * row + 1] = total;
    }
  }
  // the next segment that has tiles
  at = start + last;
  if (at >= end) return;
  if (++part_head == heads) {
    before = at;
    part_head = 0;
    do {
      if (++b == a.batch) return;
    } while (CacheTiles(a, b).count == 0);
  }
  __syncthreads();
  }
}

// Joins the parts of rows, where their segments have several; zeros where they have no tiles. A row is a wave's where there
// are many, a workgroup's where there are few; 16 lanes take a part at a time.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(kThreads) void kv4_join_kernel(const AttendArgs a) {
  __shared__ __align__(16) float numbers[16][D];
  __shared__ float stats[16][2];
  const int tid = threadIdx.x, wave = tid >> 6, g = tid / 16, d0 = tid % 16 * (D / 16);
  const int id = WAVES == 4 ? blockIdx.x : 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(wave);
  const int Q = a.queries, query = id % Q, bh = id / Q;
  const int b = min(bh / a.q_heads, a.batch - 1), head = bh % a.q_heads, G = a.q_heads / a.cache.heads;
  const bool there = bh / a.q_heads < a.batch;
  const int row = head % G * Q + query, part_head = head / G * a.rows + row / kRows;
  const Shares share = shares(a, -1, b);
  int parts = 0;
  int64_t slot = 0;
  if (share.count == 0) {
  } else if (share.whole) {
    const int64_t start = share.before + (int64_t)part_head * share.count, w0 = quotient(start, share.per);
    parts = (int)(quotient(start + share.count - 1, share.per) - w0) + 1;
    slot = w0 + (int64_t)b * a.cache.heads * a.rows + part_head;
  } else {
    slot = share.before + (int64_t)part_head * share.pieces();
    parts = (share.count + share.piece() - 1) / share.piece();
  }
  if (!there) parts = 1;
  const float* const from = a.part + slot * (kRows * (D + 2));
  const int r = row % kRows;
  float y[D / 16] = {}, top = -INFINITY, total = 0.f;
  if (parts > 1) {
#pragma unroll 4
    for (int i = g % (4 * WAVES); i < parts; i += 4 * WAVES) {
      const float* p = from + (int64_t)i * (kRows * (D + 2));
      const float t = p[kRows * D + 2 * r], sum = p[kRows * D + 2 * r + 1];
      f32x4_t x[D / 64];
#pragma unroll
      for (int e = 0; e < D / 64; ++e) x[e] = *(const f32x4_t*)(p + r * D + d0 + 4 * e);
      const float next = fmaxf(top, t), base = next == -INFINITY ? 0.f : next;
      const float f0 = exp2_raw(top - base), f1 = exp2_raw(t - base);
      top = next;
      total = total * f0 + sum * f1;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) y[e] = y[e] * f0 + x[e / 4][e % 4] * f1;
    }
  }
#pragma unroll
  for (int e = 0; e < D / 16; ++e) numbers[g][d0 + e] = y[e];
  if (d0 == 0) {
    stats[g][0] = top;
    stats[g][1] = total;
  }
  __syncthreads();
  if (parts == 1) return;  // written by its workgroup, or no row
  const int lane = WAVES == 4 ? tid : tid & 63, g0 = WAVES == 4 ? 0 : 4 * wave;
  if (lane >= D / 2) return;
  top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4 * WAVES; ++i) top = fmaxf(top, stats[g0 + i][0]);
  const float base = top == -INFINITY ? 0.f : top;
  total = 0.f;
  float y0 = 0.f, y1 = 0.f;
#pragma unroll
  for (int i = 0; i < 4 * WAVES; ++i) {
    const float f = exp2_raw(stats[g0 + i][0] - base);
    total = __builtin_fmaf(f, stats[g0 + i][1], total);
    y0 = __builtin_fmaf(f, numbers[g0 + i][2 * lane], y0);
    y1 = __builtin_fmaf(f, numbers[g0 + i][2 * lane + 1], y1);
  }
  const float f = total != 0.f ? 1.f / total : 0.f;
  ((uint32_t*)a.o.at(b, head, query))[lane] = total != 0.f ? pack2<T>(y0 * f, y1 * f) : 0u;
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

int page_shift(int64_t page) { return (page & (page - 1)) == 0 ? __builtin_ctzll((unsigned long long)page) : -1; }

int check_rows(const char* what, const char* name, const pkm_heads_t* x) {
  PKM_REQUIRE(x != nullptr && x->data != nullptr, PKM_ERR_INVALID_ARGUMENT, "%s: %s is NULL", what, name);
  PKM_REQUIRE(((uintptr_t)x->data & 15) == 0 && x->batch % 8 == 0 && x->head % 8 == 0 && x->token % 8 == 0 &&
                  x->batch >= 0 && x->head >= 0 && x->token >= 0,
              PKM_ERR_UNSUPPORTED, "%s: %s needs 16-byte aligned data and strides >= 0 that are multiples of 8", what,
              name);
  return PKM_OK;
}

Heads heads(const pkm_heads_t* x) { return {(uint8_t*)x->data, x->batch, x->head, x->token}; }

constexpr int64_t kMaxBlocks = (1ll << 32) / kThreads - 1;  // a launch takes fewer than 2^32 threads

// lanes: that work on one vector
int store_args(const char* what, StoreArgs* a, int lanes, const pkm_heads_t* k, const pkm_heads_t* v,
               const int32_t* table, int64_t width, const int32_t* starts, const int32_t* counts, int64_t batch,
               int64_t tokens) {
  int rc;
  if ((rc = check_rows(what, "k", k)) || (rc = check_rows(what, "v", v))) return rc;
  PKM_REQUIRE(starts != nullptr && counts != nullptr && (table != nullptr || width == 0), PKM_ERR_INVALID_ARGUMENT,
              "%s: table, starts and counts have to be given", what);
  PKM_REQUIRE(tokens < (1ll << 30) / a->cache.heads && batch < (1ll << 30) / a->cache.heads / tokens &&
                  2 * batch * tokens * a->cache.heads <= kMaxBlocks * (kThreads / lanes),
              PKM_ERR_UNSUPPORTED, "%s: too many tokens", what);
  a->k = heads(k), a->v = heads(v);
  a->table = table, a->starts = starts, a->counts = counts, a->width = width;
  a->batch = (int)batch, a->tokens = (int)tokens;
  a->shift = page_shift(a->cache.page);
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

// Below 2^25 tiles a sequence; query rows, each of which may need a workgroup beside the kGroups, as one launch takes.
bool attend_sizes_fit(int64_t batch, int64_t q_heads, int64_t queries, int64_t width, int64_t page) {
  const int64_t most = kMaxBlocks - kGroups;
  return width < (1ll << 30) / page && batch < most && q_heads < most && queries < most && batch * q_heads < most &&
         batch * q_heads * queries < most;
}

// Shares of a call, from sizes alone: as many workgroups as run at once, none with fewer than 4 tiles, one a wave (250
// tokens: 9.6 us against 12 with two a wave; the same from 1000 on). Cut segment by
// segment, up to one more a segment may be needed; those that are not end at once. 768: three on each of 256 CUs (512, 1024
// and 1536 took 183, 209 and 185 us where 768 took 178, and 42, 45 and 48 for one long sequence's 40).
int attend_groups(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t queries, int64_t width, int64_t page,
                  int64_t window, int64_t sinks, int64_t* segments) {
  const int64_t rows = (q_heads / kv_heads * queries + kRows - 1) / kRows;
  int64_t most = (width * page + kTok - 1) / kTok;
  if (window > 0) {
    const int64_t far = 1ll << 40;  // as good as any longer one
    const int64_t seen = (std::min(window, far) + queries) / kTok + 2 + (std::min(sinks, far) + kTok - 1) / kTok;
    if (seen < most) most = seen;
  }
  *segments = batch * kv_heads * rows;
  // (a product of large sizes may not fit; more than kGroups is all that counts)
  const double tiles = (double)*segments * (double)most;
  return tiles >= 4.0 * kGroups ? kGroups : (int)(tiles / 4.0) + 1;
}

int64_t part_bytes(int64_t groups, int64_t segments, int64_t dim) {
  return (groups + segments) * kRows * (dim + 2) * (int64_t)sizeof(float);
}

template <typename T, int D>
void launch_attend(const AttendArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)(a.groups + a.batch * a.cache.heads * a.rows);
  kv4_attend_kernel<T, D><<<grid, kThreads, 0, st>>>(a);
  const unsigned rows = (unsigned)(a.batch * a.q_heads * a.queries);
  if (rows >= 512) {
    kv4_join_kernel<T, D, 1><<<(rows + 3) / 4, kThreads, 0, st>>>(a);
  } else {
    kv4_join_kernel<T, D, 4><<<rows, kThreads, 0, st>>>(a);
  }
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
  if ((rc = store_args(what, &a, (int)dim / 32, k, v, table, width, starts, counts, batch, tokens))) return rc;
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
  if ((rc = store_args(what, &a, (int)dim / 8, k, v, table, width, starts, counts, batch, tokens))) return rc;
  return run_store<false>(what, a, dim, dtype, stream);
}

extern "C" size_t pkm_kv4_attend_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t queries,
                                                int64_t dim, int64_t width, int64_t page, int64_t window,
                                                int64_t sinks) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || queries <= 0 || dim <= 0 || dim > 128 || width < 0 || page <= 0 ||
      window < 0 || sinks < 0 || !attend_sizes_fit(batch, q_heads, queries, width, page))
    return 0;
  int64_t segments;
  const int groups = attend_groups(batch, q_heads, kv_heads, queries, width, page, window, sinks, &segments);
  return (size_t)part_bytes(groups, segments, dim);
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
  PKM_REQUIRE(attend_sizes_fit(batch, q_heads, queries, width, page), PKM_ERR_UNSUPPORTED,
              "%s: too many tokens or rows", what);
  int64_t segments;
  a.groups = attend_groups(batch, q_heads, kv_heads, queries, width, page, window, sinks, &segments);
  a.rows = (int)(segments / batch / kv_heads);
  a.cut = (int)std::max<int64_t>({1, a.groups / 4, a.groups - segments / 2});
  PKM_REQUIRE(workspace != nullptr && workspace_bytes >= (size_t)part_bytes(a.groups, segments, dim), PKM_ERR_WORKSPACE,
              "%s: workspace too small", what);
  PKM_REQUIRE(((uintptr_t)workspace & 15) == 0, PKM_ERR_INVALID_ARGUMENT, "%s: workspace is not 16-byte aligned", what);
  a.q = heads(q), a.o = heads(out);
  a.table = table, a.lengths = lengths, a.part = (float*)workspace, a.width = width;
  a.batch = (int)batch, a.q_heads = (int)q_heads, a.queries = (int)queries;
  const int64_t far = 1 << 30;
  a.window = (int)(window < far ? window : 0), a.sinks = (int)(sinks < far ? sinks : far);
  a.scale = scale;
  a.shift = page_shift(page);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKM_DTYPE_BF16) {
    dim == 128 ? launch_attend<bf16_t, 128>(a, st) : launch_attend<bf16_t, 64>(a, st);
  } else {
    dim == 128 ? launch_attend<f16_t, 128>(a, st) : launch_attend<f16_t, 64>(a, st);
  }
  return pkm_check_launch(what);
}
