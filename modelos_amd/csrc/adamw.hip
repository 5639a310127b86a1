// An AdamW step over many tensors at once, gfx950.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  g = grad * grad_scale
//   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// All arithmetic is float32; the states are held as float32, or in 8 bits: m and r = sqrt(v) as e4m3 numbers times a
// float32 step for each 256 of a tensor's numbers, step = max / 448 (e4m3's largest). r, not v, because 8 bits hold its
// range: v's exponents are twice r's. A number a >= 0 in units of its step, 2^e <= a < 2^(e + 1), e >= -6, becomes
// floor(a 2^(3 - e) + u) 2^(e - 3): rounded up or down with a dither u in [0, 1) that runs evenly through all values over
// the steps, so that what a step adds below a code's spacing is not lost on average. Nearest rounding would lose it every time:
// with b2 = 0.999 a root falls by 0.05 % of itself a step, half a spacing is 3 to 6 %. r > 0 stays above 0
// (2^-9 at least), or m would be divided by nothing.
//
// Every number is read once and written once: the step is bound by memory. 361 M bf16 numbers with masters in 127 tensors:
// 1.74 ms (5.8 TB/s); 2^30 bf16 numbers with states in 8 bits 1.78 ms (6.0 TB/s, 50 vector operations a number, which take as
// long: with 65 it was 1.96). A workgroup takes 4096 numbers of one tensor; the tensors' pointers travel in the kernel's
// arguments (48 tensors a launch), so a step copies nothing to the device.
#include "pkm_common.h"

namespace pkm {
namespace {

constexpr int kTensors = 48;  // of a launch: 72 bytes each of the 4 KB of arguments
constexpr int kChunk = 4096;  // numbers of a workgroup: 256 threads, 16 each
constexpr int kSteps = 256;   // step counters of a launch of the first kernel
constexpr int kBlock = 256;   // numbers that share a step
constexpr float kTop = 448.f; // e4m3's largest number
constexpr float kFlush = 0x1p-110f;  // a block whose largest number is below is held as zeros: 448 / max stays finite

struct Tensor {
  void* p;
  const void* g;
  void* m;  // float32, or e4m3 codes
  void* v;  // float32, or e4m3 codes of r
  float* ms;
  float* vs;
  float* master;
  const float* coefs;
  int64_t n;
};
struct Table {
  Tensor t[kTensors];
  int32_t begin[kTensors + 1];  // each tensor's first workgroup
  int32_t count;
};
struct StepTable {
  float* step[kSteps];
  int32_t count;
};

struct Coefs {
  float decay, rate, root, t;  // 1 - lr decay, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), t
};

// Counts the steps on and works out what depends on them, in 64 bits: on the device, so that a captured step counts on as well.
__global__ void adamw_begin_kernel(StepTable table, double lr, const float* lr_device, double b1, double b2, double decay,
                                   Coefs* coefs) {
  const int i = threadIdx.x;
  if (i >= table.count) return;
  const float t = *table.step[i] + 1.f;
  *table.step[i] = t;
  const double rate = lr_device ? (double)*lr_device : lr;
  coefs[i] = Coefs{(float)(1.0 - rate * decay), (float)(rate / (1.0 - pow(b1, (double)t))),
                   (float)(1.0 / sqrt(1.0 - pow(b2, (double)t))), t};
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (__is_same(T, bf16_t)) {
    return bf16_to_f32(x.x);
  } else {
    return (float)x;
  }
}
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (__is_same(T, bf16_t)) {
    return bf16_t{(uint16_t)f32_to_bf16_bits(x)};
  } else {
    return (T)x;
  }
}

// 16 and 8 bytes; NT: past the caches (non-temporal), for tensors that do not fit them.
template <bool NT>
__device__ __forceinline__ uint4 get16(const void* p) {
  return NT ? ld16_nt(p) : ld16(p);
}
template <bool NT>
__device__ __forceinline__ void put16(void* p, const uint4& v) {
  if constexpr (NT) {
    st16_nt((uint4*)p, v);
  } else {
    st16(p, v);
  }
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <bool NT>
__device__ __forceinline__ u32x2 get8(const void* p) {
  return NT ? __builtin_nontemporal_load((const u32x2*)p) : *(const u32x2*)p;
}
template <bool NT>
__device__ __forceinline__ void put8(void* p, u32x2 v) {
  if constexpr (NT) {
    __builtin_nontemporal_store(v, (u32x2*)p);
  } else {
    *(u32x2*)p = v;
  }
}

// How a thread reaches its numbers: WIDE: in whole vectors, all of which exist; else one by one, as far as they do.
template <bool WIDE_, bool NT_>
struct Access {
  static constexpr bool WIDE = WIDE_, NT = NT_;
};

// N numbers at x + i, of which those below n exist.
template <typename T, int N, typename A>
__device__ __forceinline__ void load_n(const T* x, int64_t i, int64_t n, float* f) {
  if constexpr (!A::WIDE) {
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = i + k < n ? to_float(x[i + k]) : 0.f;
  } else if constexpr (N * sizeof(T) == 8) {
    const u32x2 w = get8<A::NT>(x + i);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = to_float(__builtin_bit_cast(T, (uint16_t)(w[k / 2] >> (k % 2 * 16))));
  } else {
    constexpr int E = VecTraits<T>::EPV;
#pragma unroll
    for (int k = 0; k < N / E; ++k) VecTraits<T>::unpack(get16<A::NT>(x + i + k * E), f + k * E);
  }
}
template <typename T, int N, typename A>
__device__ __forceinline__ void store_n(T* x, int64_t i, int64_t n, const float* f) {
  if constexpr (!A::WIDE) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k < n) x[i + k] = from_float<T>(f[k]);
  } else if constexpr (N * sizeof(T) == 8) {
    u32x2 w;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w[k] = (uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(f[2 * k])) |
             ((uint32_t)__builtin_bit_cast(uint16_t, from_float<T>(f[2 * k + 1])) << 16);
    put8<A::NT>(x + i, w);
  } else {
    constexpr int E = VecTraits<T>::EPV;
#pragma unroll
    for (int k = 0; k < N / E; ++k) put16<A::NT>(x + i + k * E, VecTraits<T>::pack(f + k * E));
  }
}

struct Betas {
  float b1, a1, b2, a2, eps;  // a = 1 - b, rounded once
};

__device__ __forceinline__ float updated(float p, float m, float root_v, const Coefs& c, float eps) {
  // v_rcp_f32 and v_sqrt_f32 are within an ulp: of the step, not of the weight
  return p * c.decay - c.rate * m * __builtin_amdgcn_rcpf(root_v * c.root + eps);
}

// Largest of the lanes' bits among 32 lanes; bits of numbers >= 0 order as the numbers do, NaN above all.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float max32(uint32_t x) {
  x = dpp_max<0xB1>(x);   // quad_perm [1,0,3,2]
  x = dpp_max<0x4E>(x);   // quad_perm [2,3,0,1]
  x = dpp_max<0x141>(x);  // row_half_mirror
  x = dpp_max<0x140>(x);  // row_mirror
  return __uint_as_float(max(x, (uint32_t)__builtin_amdgcn_ds_swizzle((int)x, 0x401F)));  // lane xor 16
}

// The code of a >= 0 (units of the step) in the upper byte, from 2^-120 a and the dither in the low 20 bits of u. 2^-120 a
// has e4m3's exponents as a float32: its bits above bit 20 count e4m3's numbers from 0 on, the smallest ones among them, as
// float32's own smallest numbers are spaced evenly too. So adding the dither below them rounds. The float32 is a product with
// the step's reciprocal, a few units of its last place off x / step: where the sum comes within 8 of a code's border, `near`
// falls below kNear and exact_code() decides. (A code past the largest, 448 and a little, is such a case.)
constexpr uint32_t kNear = 16u << 12;
__device__ __forceinline__ uint32_t code_of(float a, uint32_t u, uint32_t& near) {
  const uint32_t code = (__float_as_uint(a) + u) << 4;
  near = min(near, (code << 8) + kNear / 2);
  return code;
}
// The upper bytes of four.
__device__ __forceinline__ uint32_t upper_bytes(const uint32_t* c) {
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0703u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0703u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// The same of x / step, not rounded: x is compared with the border nearest to it, times the step, in one exact sign.
__device__ __forceinline__ uint32_t exact_code(float x, float step, uint32_t u) {
  const float a = x / step;
  const bool small = a < 0x1p-6f;
  const uint32_t bits = __float_as_uint(small ? a + 0x1p-6f : a) + u;
  const uint32_t high = (bits + 0x80000u) >> 20;  // the code above the nearest border
  const float at = __uint_as_float((high << 20) - u);
  const float border = small ? at - 0x1p-6f : at;
  const float up = step < 0x1p-60f ? 0x1p60f : 1.f;  // so that no difference is below float32's smallest numbers
  const uint32_t code = high - (__builtin_fmaf(border, step * up, -x * up) > 0.f ? 1u : 0u) - (small ? (121u << 3) : (120u << 3));
  return code < 0x7eu ? code : 0x7eu;
}

// States of 8 bits: twice eight numbers in a row a thread, 2048 apart; the 32 lanes of a block of 256 side by side.
template <typename T, bool MASTER, typename A>
__device__ __forceinline__ void step8(const Tensor& x, int64_t first, int64_t n, const Coefs& c, const Betas& b, float gs,
                                      bool scaled) {
#pragma clang fp contract(off)  // each operation rounded but for the two written as one: states that do not hang on the build
  float p[2][8], g[2][8], steps[2][2];
  uint32_t codes[2][2][2];  // [numbers][m, r][words]
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t i = first + k * 2048;
    if constexpr (MASTER) {
      load_n<float, 8, A>(x.master, i, n, p[k]);
    } else {
      load_n<T, 8, A>((const T*)x.p, i, n, p[k]);
    }
    load_n<T, 8, A>((const T*)x.g, i, n, g[k]);
    const int64_t block = min(i, n - 1) / kBlock;
    steps[k][0] = x.ms[block];
    steps[k][1] = x.vs[block];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* const from = (const uint8_t*)(s ? x.v : x.m) + i;
      if constexpr (A::WIDE) {
        const u32x2 w = get8<A::NT>(from);
        codes[k][s][0] = w[0];
        codes[k][s][1] = w[1];
      } else {
        codes[k][s][0] = codes[k][s][1] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < n) codes[k][s][e / 4] |= (uint32_t)from[e] << (e % 4 * 8);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t i = first + k * 2048;
    float m[8], v[8], root[8];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const auto m0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[k][0][w], false),
                 m1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[k][0][w], true);
      const auto v0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[k][1][w], false),
                 v1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[k][1][w], true);
      m[4 * w] = m0[0], m[4 * w + 1] = m0[1], m[4 * w + 2] = m1[0], m[4 * w + 3] = m1[1];
      v[4 * w] = v0[0], v[4 * w + 1] = v0[1], v[4 * w + 2] = v1[0], v[4 * w + 3] = v1[1];
    }
    if (scaled) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[k][e] *= gs;
    }
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = g[k][e], r = v[e] * steps[k][1];
      m[e] = __builtin_fmaf(b.a1, ge, b.b1 * (m[e] * steps[k][0]));
      v[e] = __builtin_fmaf(b.a2, ge * ge, b.b2 * (r * r));
      root[e] = __builtin_amdgcn_sqrtf(v[e]);
      p[k][e] = updated(p[k][e], m[e], root[e], c, b.eps);
      if constexpr (MASTER) asm("" : "+v"(p[k][e]));  // the weight rounds the master, not the operation before it
      top_m = max(top_m, __float_as_uint(m[e]) & 0x7fffffffu);
      top_v = max(top_v, __float_as_uint(v[e]));
    }
    if constexpr (MASTER) store_n<float, 8, A>(x.master, i, n, p[k]);
    store_n<T, 8, A>((T*)x.p, i, n, p[k]);
    // the root's rounding keeps the order: the largest root is the largest's root
    const float mm = max32(top_m), mr = sqrtf(max32(top_v));
    const bool no_m = mm < kFlush, no_r = mr < kFlush;
    // 2^-120 / step, as long as that is one of float32's full numbers; exact_code() serves larger blocks
    const float fm = no_m ? 0.f : kTop * 0x1p-120f * __builtin_amdgcn_rcpf(mm);
    const float fr = no_r ? 0.f : kTop * 0x1p-120f * __builtin_amdgcn_rcpf(mr);
    const uint32_t least = no_r ? 0u : 1u << 24;
    const float step_m = no_m ? 0.f : mm * (1.f / kTop), step_r = no_r ? 0.f : mr * (1.f / kTop);
    if ((threadIdx.x & 31) == 0 && i < n) {
      x.ms[i / kBlock] = step_m;
      x.vs[i / kBlock] = step_r;
    }
    const uint32_t u0 = (uint32_t)i * 2654435761u + (uint32_t)c.t * 2246822519u;
    // v_sqrt_f32 is not exact enough below 2^-126, where the smallest roots of a block of roots up to 2^-43 come from
    const bool far_off = max(mm, mr) > kTop * 0x1p6f || (mr < 0x1p-43f && !no_r);
    uint32_t cm[2], cr[2], near = far_off ? 0u : ~0u, u = u0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint32_t a[4], d[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = code_of(fabsf(m[4 * w + e]) * fm, u >> 12, near) | (__float_as_uint(m[4 * w + e]) & 0x80000000u);
        // a root above 0 is above 2^-75: `least`, the code 1, or 0
        d[e] = max(code_of(root[4 * w + e] * fr, u & 0xfffffu, near), min(__float_as_uint(root[4 * w + e]), least));
        u += 2654435761u;
      }
      cm[w] = upper_bytes(a);
      cr[w] = upper_bytes(d);
    }
    if (near < kNear) {  // one lane in 4000
      u = u0;
      cm[0] = cm[1] = cr[0] = cr[1] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t a = no_m ? 0u : exact_code(fabsf(m[e]), step_m, u >> 12);
        const float r = sqrtf(v[e]);
        const uint32_t d = no_r ? 0u : max(exact_code(r, step_r, u & 0xfffffu), r > 0.f ? 1u : 0u);
        cm[e / 4] |= (a | ((__float_as_uint(m[e]) >> 24) & 0x80u)) << (e % 4 * 8);
        cr[e / 4] |= d << (e % 4 * 8);
        u += 2654435761u;
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint8_t* const to = (uint8_t*)(s ? x.v : x.m) + i;
      const uint32_t* const w = s ? cr : cm;
      if constexpr (A::WIDE) {
        put8<A::NT>(to, u32x2{w[0], w[1]});
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < n) to[e] = (uint8_t)(w[e / 4] >> (e % 4 * 8));
      }
    }
  }
}

// States of 32 bits: four times four numbers a thread, 1024 apart, so that every access of a wave is one stretch of memory,
// in 16 bits and in 32.
template <typename T, bool MASTER, typename A>
__device__ __forceinline__ void step32(const Tensor& x, int64_t first, int64_t n, const Coefs& c, const Betas& b, float gs) {
#pragma clang fp contract(off)
  float p[4][4], g[4][4], m[4][4], v[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = first + k * 1024;
    if constexpr (MASTER) {
      load_n<float, 4, A>(x.master, i, n, p[k]);
    } else {
      load_n<T, 4, A>((const T*)x.p, i, n, p[k]);
    }
    load_n<T, 4, A>((const T*)x.g, i, n, g[k]);
    load_n<float, 4, A>((const float*)x.m, i, n, m[k]);
    load_n<float, 4, A>((const float*)x.v, i, n, v[k]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = first + k * 1024;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g[k][e] *= gs;
      m[k][e] = __builtin_fmaf(b.a1, g[k][e], b.b1 * m[k][e]);
      v[k][e] = __builtin_fmaf(b.a2, g[k][e] * g[k][e], b.b2 * v[k][e]);
      p[k][e] = updated(p[k][e], m[k][e], __builtin_amdgcn_sqrtf(v[k][e]), c, b.eps);
      if constexpr (MASTER) asm("" : "+v"(p[k][e]));  // the weight rounds the master, not the operation before it
    }
    if constexpr (MASTER) store_n<float, 4, A>(x.master, i, n, p[k]);
    store_n<T, 4, A>((T*)x.p, i, n, p[k]);
    store_n<float, 4, A>((float*)x.m, i, n, m[k]);
    store_n<float, 4, A>((float*)x.v, i, n, v[k]);
  }
}

template <typename T, int BITS, bool MASTER, bool NT>
__global__ __launch_bounds__(256) void adamw_kernel(Table table, Betas b, const float* grad_scale) {
  int at = 0;  // the last tensor that begins at or before this workgroup
  for (int s = 32; s > 0; s >>= 1)
    if (at + s < table.count && table.begin[at + s] <= (int)blockIdx.x) at += s;
  const Tensor& x = table.t[at];
  const int64_t first = (int64_t)((int)blockIdx.x - table.begin[at]) * kChunk, n = x.n;
  const Coefs c = *(const Coefs*)x.coefs;
  const float gs = grad_scale ? *grad_scale : 1.f;
  const uintptr_t all = (uintptr_t)x.p | (uintptr_t)x.g | (uintptr_t)x.m | (uintptr_t)x.v | (uintptr_t)x.master;
  // whole vectors where every pointer allows them and the workgroup is full
  const bool wide = (all & 15) == 0 && first + kChunk <= n;
  if constexpr (BITS == 32) {
    const int64_t i = first + threadIdx.x * 4;
    if (wide) {
      step32<T, MASTER, Access<true, NT>>(x, i, n, c, b, gs);
    } else {
      step32<T, MASTER, Access<false, false>>(x, i, n, c, b, gs);
    }
  } else {
    const int64_t i = first + threadIdx.x * 8;
    if (wide) {
      step8<T, MASTER, Access<true, NT>>(x, i, n, c, b, gs, grad_scale != nullptr);
    } else {
      step8<T, MASTER, Access<false, false>>(x, i, n, c, b, gs, grad_scale != nullptr);
    }
  }
}

template <typename T, int BITS, bool MASTER>
void launch(const Table& table, bool nt, unsigned blocks, const Betas& b, const float* gs, hipStream_t st) {
  if (nt)
    hipLaunchKernelGGL((adamw_kernel<T, BITS, MASTER, true>), dim3(blocks), dim3(256), 0, st, table, b, gs);
  else
    hipLaunchKernelGGL((adamw_kernel<T, BITS, MASTER, false>), dim3(blocks), dim3(256), 0, st, table, b, gs);
}
template <typename T>
void launch(const Table& table, int bits, bool master, unsigned blocks, const Betas& b, const float* gs, hipStream_t st) {
  // What a launch touches: past the caches if it is more than the 256 MB they hold. 361 M numbers, bf16 with masters: 1.74 ms
  // so, 1.88 through them; 1.8 M float32 numbers, touched again each step: 9.7 us so, 6.5 to 8 through them.
  const int64_t bytes = (int64_t)blocks * kChunk * ((int64_t)sizeof(T) * 2 + (bits == 32 ? 8 : 2) + (master ? 4 : 0));
  const bool nt = bytes > (256ll << 20);
  if (bits == 32)
    master ? launch<T, 32, true>(table, nt, blocks, b, gs, st) : launch<T, 32, false>(table, nt, blocks, b, gs, st);
  else
    master ? launch<T, 8, true>(table, nt, blocks, b, gs, st) : launch<T, 8, false>(table, nt, blocks, b, gs, st);
}

}  // namespace
}  // namespace pkm

using namespace pkm;

extern "C" size_t pkm_adamw_workspace_size(int64_t count) {
  return count > 0 && count < (1ll << 31) ? (size_t)count * sizeof(Coefs) : 0;
}

extern "C" int pkm_adamw_step(const pkm_adamw_tensor_t* tensors, int64_t count, int dtype, int state_bits, double lr,
                              const float* lr_device, double beta1, double beta2, double eps, double weight_decay,
                              const float* grad_scale, void* workspace, size_t workspace_bytes, void* stream) {
  PKM_REQUIRE(count >= 0 && count < (1ll << 31), PKM_ERR_INVALID_ARGUMENT, "pkm_adamw_step: %lld tensors", (long long)count);
  PKM_REQUIRE(dtype == PKM_DTYPE_F32 || dtype == PKM_DTYPE_BF16 || dtype == PKM_DTYPE_F16, PKM_ERR_INVALID_ARGUMENT,
              "pkm_adamw_step: dtype %d", dtype);
  PKM_REQUIRE(state_bits == 32 || state_bits == 8, PKM_ERR_INVALID_ARGUMENT, "pkm_adamw_step: states of %d bits (32 or 8)",
              state_bits);
  if (count == 0) return PKM_OK;
  PKM_REQUIRE(tensors, PKM_ERR_INVALID_ARGUMENT, "pkm_adamw_step: null pointer");
  bool any = false, master = false;  // of the tensors that have numbers
  for (int64_t i = 0; i < count; ++i) {
    const pkm_adamw_tensor_t& t = tensors[i];
    PKM_REQUIRE(t.numel >= 0, PKM_ERR_INVALID_ARGUMENT, "pkm_adamw_step: tensor %lld has a negative size", (long long)i);
    PKM_REQUIRE(t.numel < (1ll << 35), PKM_ERR_UNSUPPORTED,
                "pkm_adamw_step: tensor %lld has %lld numbers (fewer than 2^35 are supported)", (long long)i, (long long)t.numel);
    PKM_REQUIRE(t.step, PKM_ERR_INVALID_ARGUMENT, "pkm_adamw_step: tensor %lld has no step counter", (long long)i);
    if (t.numel == 0) continue;
    PKM_REQUIRE(t.param && t.grad && t.exp_avg && t.second, PKM_ERR_INVALID_ARGUMENT,
                "pkm_adamw_step: tensor %lld has a null pointer", (long long)i);
    PKM_REQUIRE(state_bits == 32 || (t.exp_avg_scale && t.second_scale), PKM_ERR_INVALID_ARGUMENT,
                "pkm_adamw_step: tensor %lld has no steps", (long long)i);
    PKM_REQUIRE(!any || (t.master != nullptr) == master, PKM_ERR_INVALID_ARGUMENT,
                "pkm_adamw_step: all tensors have masters or none has");
    any = true;
    master = t.master != nullptr;
  }
  PKM_REQUIRE(workspace && workspace_bytes >= pkm_adamw_workspace_size(count), PKM_ERR_WORKSPACE,
              "pkm_adamw_step: workspace of %zu bytes, %zu needed", workspace_bytes, pkm_adamw_workspace_size(count));
  PKM_REQUIRE(((uintptr_t)workspace & 15) == 0, PKM_ERR_INVALID_ARGUMENT, "pkm_adamw_step: workspace not 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  Coefs* coefs = (Coefs*)workspace;
  for (int64_t i = 0; i < count; i += kSteps) {
    StepTable steps;
    steps.count = (int32_t)(count - i < kSteps ? count - i : kSteps);
    for (int k = 0; k < steps.count; ++k) steps.step[k] = tensors[i + k].step;
    hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(kSteps), 0, st, steps, lr, lr_device, beta1, beta2, weight_decay,
                       coefs + i);
  }
  const Betas betas{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
  Table table;
  int64_t blocks = 0;
  table.count = 0;
  auto flush = [&]() {
    if (table.count == 0) return;
    if (dtype == PKM_DTYPE_F32)
      launch<float>(table, state_bits, master, (unsigned)blocks, betas, grad_scale, st);
    else if (dtype == PKM_DTYPE_BF16)
      launch<bf16_t>(table, state_bits, master, (unsigned)blocks, betas, grad_scale, st);
    else
      launch<f16_t>(table, state_bits, master, (unsigned)blocks, betas, grad_scale, st);
    table.count = 0;
    blocks = 0;
  };
  for (int64_t i = 0; i < count; ++i) {
    const pkm_adamw_tensor_t& t = tensors[i];
    if (t.numel == 0) continue;
    const int64_t more = (t.numel + kChunk - 1) / kChunk;
    if (table.count == kTensors || blocks + more >= (1ll << 24)) flush();  // fewer than 2^32 threads a launch
    table.t[table.count] = Tensor{t.param, t.grad, t.exp_avg, t.second, t.exp_avg_scale, t.second_scale, t.master,
                                  (const float*)(coefs + i), t.numel};
    table.begin[table.count++] = (int32_t)blocks;
    blocks += more;
  }
  flush();
  return pkm_check_launch("pkm_adamw_step");
}
