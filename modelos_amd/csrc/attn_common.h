// Shared pieces of the attention kernels (gfx950 / CDNA4, wave64): matrix
// instruction types, the LDS tile layout and its loads.
//
// Matrix operand layouts (lane = 32 h + l for 32x32x16, 16 q + l for 16x16x32):
//   A [rows, k], B [k, cols]: row / col l, k = 8 h + j (8 q + j), j = 0..7
//   C [rows, cols], 32x32:    col l, row 8 (i / 4) + 4 h + i % 4, i = 0..15
//   C [rows, cols], 16x16:    col l, row 4 q + i, i = 0..3
// The order of k is free as long as both operands share it. A C tile rounded
// to 16 bits is the B operand of the next product with its rows as k: element
// i of 16 becomes k step i / 8, element i % 8, that is row
// 16 (i / 8) + 8 (i % 8 / 4) + 4 h + i % 4. The A operand beside it is read from
// LDS in that order (frag_cols).
#pragma once

#include "pkm_common.h"

namespace pkm {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// 8 numbers of 16 bits, one matrix operand register set
typedef u32x4_t frag_t;

template <typename T>
__device__ __forceinline__ f32x16_t mfma32(frag_t a, frag_t b, f32x16_t c) {
  if constexpr (sizeof(T) == 2 && __is_same(T, bf16_t)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
}

template <typename T>
__device__ __forceinline__ f32x4_t mfma16(frag_t a, frag_t b, f32x4_t c) {
  if constexpr (__is_same(T, bf16_t)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
}

// Two floats to a packed pair of T, round to nearest even.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (__is_same(T, bf16_t)) {
    return pack2_bf16(lo, hi);
  } else {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
  }
}

template <typename T>
__device__ __forceinline__ float unpack1(uint32_t bits) {
  if constexpr (__is_same(T, bf16_t)) {
    return bf16_to_f32(bits);
  } else {
    return f16_bits_to_f32(bits);
  }
}

// v_exp_f32 (results under 2^-126 are 0)
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// The other half wave's value: lane 32 h + l gets that of lane 32 (1 - h) + l.
__device__ __forceinline__ float swap_halves(float x) {
  const u32x2_t r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                                               false, false));
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// ---------------------------------------------------------------------------
// A tile of rows of D 16-bit numbers in LDS. The 16-byte chunks of a row are
// permuted by xor with swizzle(row), so that neither 16 rows read at one chunk
// (frag_rows) nor 4 rows read at 4 chunks (frag_cols) share banks.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4;
typedef __attribute__((address_space(3))) f32x4_t lds_f32x4;

template <int D>
__device__ __forceinline__ int tile_offset(int row, int chunk) {
  const int f = D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  return row * (D * 2) + ((chunk ^ f) << 4);
}

// Where a lane's operands lie in a tile: the first k step's (rows_at) and the first 32 columns' (cols_at). The others
// are an xor away, as the permutation is one: tiles start at multiples of 256 bytes.
template <int D>
__device__ __forceinline__ uint32_t rows_at(int lane) {
  return tile_offset<D>(lane & 31, lane >> 5);
}
template <int D>
__device__ __forceinline__ uint32_t cols_at(int lane) {
  const int l = lane & 15, h = lane >> 5, g = (lane >> 4) & 1;
  return tile_offset<D>(4 * h + (l >> 2), 2 * g + ((l & 3) >> 1)) + (l & 1) * 8;
}

// A operand whose rows are the tile's rows row0 .. row0 + 31, k step s of 16 numbers. at: the tile + rows_at.
template <int D>
__device__ __forceinline__ frag_t frag_rows(uint32_t at, int row0, int s) {
  return *(const lds_u32x4*)(uintptr_t)((at ^ (uint32_t)(s << 5)) + row0 * (D * 2));
}

// A operand whose rows are the tile's columns 32 t .. 32 t + 31 and whose k are the tile's rows
// row0 + 8 (j / 4) + 4 h + j % 4 (the order of a C tile used as B operand). at: the tile + cols_at.
template <int D>
__device__ __forceinline__ frag_t frag_cols(uint32_t at, int row0, int t) {
  const uint32_t p = (at ^ (uint32_t)(t << 6)) + row0 * (D * 2), q = (at ^ (uint32_t)((t << 6) | 32)) + (row0 + 8) * (D * 2);
  const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)p);
  const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)q);
  const u32x2_t x = __builtin_bit_cast(u32x2_t, a), y = __builtin_bit_cast(u32x2_t, b);
  return (frag_t){x[0], x[1], y[0], y[1]};
}

// B operand, k step s, of rows that lie in global memory: 8 numbers of the lane's row (nullptr reads zeros).
template <int D>
__device__ __forceinline__ frag_t frag_global(const void* row, int s, int lane) {
  frag_t z = {0, 0, 0, 0};
  return row ? *(const frag_t*)((const uint8_t*)row + (2 * s + (lane >> 5)) * 16) : z;
}

// 64 lanes' 16 bytes each from a buffer at the lanes' offsets to LDS at `to` (uniform) and on, side by side. In asm,
// so that the compiler does not wait for it at the next transposing read of another tile; there is no register
// for it to lose, and tile_wait() before the barrier is the wait. The s_nop: m0 is read one state after its write, a
// descriptor that a vector instruction wrote (a lane read, a spilled scalar) five; the compiler does not see to it in here.
__device__ __forceinline__ void load_lds16(u32x4_t rsrc, lds_u8* to, uint32_t offset) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"((uint32_t)(uintptr_t)to), "v"(offset), "s"(rsrc)
               : "memory");
}

// A tile's rows from global memory straight to LDS (no registers in between), by WAVES waves. A wave's load
// writes 64 chunks of 16 bytes side by side; the permutation is in the addresses that the lanes read. Rows from
// `last` (>= 1) on repeat row last - 1: what lies behind a sequence is never read. Row 0 is the caller's: a tile that begins before
// its sequence holds what lies there. The loads are complete after tile_wait().
template <int D, int ROWS, int WAVES = 4>
struct TileLoad {
  static constexpr int CH = D / 8, PER = 64 / CH, N = ROWS / PER / WAVES;  // rows of a load, loads of a wave
  static_assert(PER * WAVES % 16 == 0 && N * PER * WAVES == ROWS, "one permutation a lane");
  int row, chunk;  // the lane's first row and its bytes within a row
  __device__ __forceinline__ TileLoad(int tid) {
    const int wave = tid >> 6, lane = tid & 63;
    row = wave * PER + lane / CH;
    // rows of one lane are WAVES PER apart, a multiple of 16: one permutation
    chunk = tile_offset<D>(row, lane % CH) - row * (D * 2);
  }
  // base: row 0 of the tile; stride in bytes (128 rows of it fit in 31 bits)
  __device__ __forceinline__ void load(lds_u8* tile, const uint8_t* base, uint32_t stride, int last, int tid) const {
    const u32x4_t rs = {(uint32_t)(uintptr_t)base, (uint32_t)((uintptr_t)base >> 32), 0x7fffffffu, 0x00020000u};
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
    for (int i = 0; i < N; ++i)
      load_lds16(rs, tile + (wave + WAVES * i) * 1024,
                 (uint32_t)min(row + WAVES * PER * i, last - 1) * stride + chunk);
  }
};
// 64 lanes' float each, as load_lds16.
__device__ __forceinline__ void load_lds4(u32x4_t rsrc, lds_u8* to, uint32_t offset) {
  asm volatile("s_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"{m0}"((uint32_t)(uintptr_t)to), "v"(offset), "s"(rsrc)
               : "memory");
}

// Waits for the wave's loads to LDS but the last N.
template <int N = 0>
__device__ __forceinline__ void tile_wait() {
  static_assert(N < 16, "the low four bits of the count");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | N);  // vmcnt(N), which the compiler's own counting sees
  asm volatile("" ::: "memory");
}

// A point that the compiler moves no LDS read and no matrix instruction across: the loops below issue the reads of
// a later product in front of each product, and its scheduler would pull them back behind it.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x0406); }

__device__ __forceinline__ uint32_t lds_address(const lds_u8* p) { return (uint32_t)(uintptr_t)p; }

// A [batch, heads, tokens, dim] tensor in a kernel's arguments, strides in elements (pkm_heads_t of the C ABI).
struct Heads {
  uint8_t* p;
  int64_t batch, head, token;
  __device__ __forceinline__ uint8_t* at(int64_t b, int64_t h, int64_t t) const {
    return p + 2 * (b * batch + h * head + t * token);
  }
};

// Row of a C^T tile set (columns = the lane's row of the tensor, rows = its numbers) times f to memory; with rest, what
// the rounding left of it there.
template <typename T, int D>
__device__ __forceinline__ void store_row(uint8_t* row, const f32x16_t (&acc)[D / 32], float f, int lane,
                                          uint8_t* rest = nullptr) {
  const int h = lane >> 5;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int at = 2 * (32 * t + 8 * a + 4 * h);
      u32x2_t x, r;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float y = acc[t][4 * a + 2 * e] * f, z = acc[t][4 * a + 2 * e + 1] * f;
        x[e] = pack2<T>(y, z);
        if (rest) r[e] = pack2<T>(y - unpack1<T>(x[e] & 0xffffu), z - unpack1<T>(x[e] >> 16));
      }
      *(u32x2_t*)(row + at) = x;
      if (rest) *(u32x2_t*)(rest + at) = r;
    }
}

}  // namespace pkm
