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
// with b2 = 0.999 a state falls by 0.05 % a step, a twentieth to an hundredth of half a spacing. r > 0 stays above 0
// (2^-9 at least), or m would be divided by nothing.
//
// Every number is read once and written once: the step is bound by memory. A workgroup takes 4096 numbers of one tensor;
// the tensors' pointers travel in the kernel's arguments (48 tensors a launch), so a step copies nothing to the device.
#include "pkm_common.h"

namespace pkm {
namespace {

constexpr int kTensors = 48;     // of a launch: 72 bytes each of the 4 KB of arguments
constexpr int kChunk = 4096;     // numbers of a workgroup: 256 threads, 16 each
constexpr int kSteps = 256;      // step counters of a launch of the first kernel
constexpr int kBlock = 256;      // numbers that share a step
constexpr float kTop = 448.f;    // e4m3's largest number
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

// N numbers at x + i, of which those below n exist; WIDE: 16-byte vectors, all of them exist.
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void load_n(const T* x, int64_t i, int64_t n, float* f) {
  if constexpr (WIDE) {
    constexpr int E = VecTraits<T>::EPV;
#pragma unroll
    for (int k = 0; k < N / E; ++k) VecTraits<T>::unpack(ld16(x + i + k * E), f + k * E);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = i + k < n ? to_float(x[i + k]) : 0.f;
  }
}
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void store_n(T* x, int64_t i, int64_t n, const float* f) {
  if constexpr (WIDE) {
    constexpr int E = VecTraits<T>::EPV;
#pragma unroll
    for (int k = 0; k < N / E; ++k) st16(x + i + k * E, VecTraits<T>::pack(f + k * E));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k < n) x[i + k] = from_float<T>(f[k]);
  }
}

struct Betas {
  float b1, a1, b2, a2, eps;  // a = 1 - b, rounded once
};

__device__ __forceinline__ float updated(float p, float m, float root_v, const Coefs& c, float eps) {
  // v_rcp_f32 and v_sqrt_f32 are within an ulp: of the step, not of the weight
  return p * c.decay - c.rate * m * __builtin_amdgcn_rcpf(root_v * c.root + eps);
}

// Largest of the lanes' bits among 16 lanes; bits of numbers >= 0 order as the numbers do, NaN above all.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
  return x > y ? x : y;
}
__device__ __forceinline__ float max16(uint32_t x) {
  x = dpp_max<0xB1>(x);
  x = dpp_max<0x4E>(x);
  x = dpp_max<0x141>(x);
  return __uint_as_float(dpp_max<0x140>(x));
}

// The code of a >= 0 (units of the step), dither in the low 20 bits of u. A float's bits above bit 20 count e4m3's numbers
// of the same exponents, so adding the dither below them rounds; under 2^-6, where the spacing stays 2^-9, so do the bits of
// a + 2^-6. `a` is a product with the step's reciprocal, a few units of its last place off x / step: where the sum comes
// within 8 of a code's border, `near` falls below 16 and exact_code() decides.
__device__ __forceinline__ uint32_t code_of(float a, uint32_t u, uint32_t& near) {
  const bool small = a < 0x1p-6f;
  const uint32_t bits = __float_as_uint(small ? a + 0x1p-6f : a) + u;
  const uint32_t code = (bits >> 20) - (small ? (121u << 3) : (120u << 3));
  near = min(near, (bits + 8) & 0xfffffu);
  return code < 0x7eu ? code : 0x7eu;
}

// The same of x / step, not rounded: x is compared with the border nearest to it, times the step, in one exact sign.
__device__ __forceinline__ uint32_t exact_code(float x, float step, float f, uint32_t u) {
  const float a = x * f;
  const bool small = a < 0x1p-6f;
  const uint32_t bits = __float_as_uint(small ? a + 0x1p-6f : a) + u;
  const uint32_t high = (bits + 0x80000u) >> 20;  // the code above the nearest border
  const float at = __uint_as_float((high << 20) - u);
  const float border = small ? at - 0x1p-6f : at;
  const uint32_t code = high - (__builtin_fmaf(border, step, -x) > 0.f ? 1u : 0u) - (small ? (121u << 3) : (120u << 3));
  return code < 0x7eu ? code : 0x7eu;
}

template <typename T, int BITS, bool MASTER, bool WIDE>
__device__ __forceinline__ void step_of(const Tensor& x, int64_t i, int64_t n, const Coefs& c, const Betas& b, float gs) {
#pragma clang fp contract(off)  // each operation rounded but for the two written as one: states that do not hang on the build
  float p[16], g[16], m[16], v[16];
  if constexpr (MASTER) {
    load_n<float, 16, WIDE>(x.master, i, n, p);
  } else {
    load_n<T, 16, WIDE>((const T*)x.p, i, n, p);
  }
  load_n<T, 16, WIDE>((const T*)x.g, i, n, g);
  float ms, vs;
  if constexpr (BITS == 32) {
    load_n<float, 16, WIDE>((const float*)x.m, i, n, m);
    load_n<float, 16, WIDE>((const float*)x.v, i, n, v);
  } else {
    const int64_t block = min(i, n - 1) / kBlock;
    ms = x.ms[block];
    vs = x.vs[block];
    uint32_t cm[4] = {}, cv[4] = {};
    if constexpr (WIDE) {
      const uint4 a = ld16((const uint8_t*)x.m + i), d = ld16((const uint8_t*)x.v + i);
      cm[0] = a.x, cm[1] = a.y, cm[2] = a.z, cm[3] = a.w;
      cv[0] = d.x, cv[1] = d.y, cv[2] = d.z, cv[3] = d.w;
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (i + k < n) {
          cm[k / 4] |= (uint32_t)((const uint8_t*)x.m)[i + k] << (k % 4 * 8);
          cv[k / 4] |= (uint32_t)((const uint8_t*)x.v)[i + k] << (k % 4 * 8);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const auto m0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)cm[k], false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)cm[k], true);
      const auto v0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)cv[k], false), v1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)cv[k], true);
      m[4 * k] = m0[0] * ms, m[4 * k + 1] = m0[1] * ms, m[4 * k + 2] = m1[0] * ms, m[4 * k + 3] = m1[1] * ms;
      v[4 * k] = v0[0] * vs, v[4 * k + 1] = v0[1] * vs, v[4 * k + 2] = v1[0] * vs, v[4 * k + 3] = v1[1] * vs;
    }
  }
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    g[k] *= gs;
    if constexpr (BITS == 8) v[k] *= v[k];
    m[k] = __builtin_fmaf(b.a1, g[k], b.b1 * m[k]);
    v[k] = __builtin_fmaf(b.a2, g[k] * g[k], b.b2 * v[k]);
    p[k] = updated(p[k], m[k], __builtin_amdgcn_sqrtf(v[k]), c, b.eps);
    if constexpr (MASTER) asm("" : "+v"(p[k]));  // the weight rounds the master, not the operation before it
    if constexpr (BITS == 8) {
      top_m = max(top_m, __float_as_uint(m[k]) & 0x7fffffffu);
      top_v = max(top_v, __float_as_uint(v[k]));
    }
  }
  if constexpr (MASTER) store_n<float, 16, WIDE>(x.master, i, n, p);
  store_n<T, 16, WIDE>((T*)x.p, i, n, p);
  if constexpr (BITS == 32) {
    store_n<float, 16, WIDE>((float*)x.m, i, n, m);
    store_n<float, 16, WIDE>((float*)x.v, i, n, v);
  } else {
    // the root's rounding keeps the order: the largest root is the largest's root
    const float mm = max16(top_m), mr = sqrtf(max16(top_v));
    const bool no_m = mm < kFlush, no_r = mr < kFlush;
    const float fm = no_m ? 0.f : kTop / mm, fr = no_r ? 0.f : kTop / mr;
    const float step_m = no_m ? 0.f : mm * (1.f / kTop), step_r = no_r ? 0.f : mr * (1.f / kTop);
    if ((threadIdx.x & 15) == 0 && i < n) {
      x.ms[i / kBlock] = step_m;
      x.vs[i / kBlock] = step_r;
    }
    const uint32_t u0 = (uint32_t)i * 2654435761u + (uint32_t)c.t * 2246822519u;
    uint32_t cm[4] = {}, cv[4] = {}, near = ~0u, u = u0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const uint32_t a = code_of(fabsf(m[k]) * fm, u >> 12, near);
      const float r = __builtin_amdgcn_sqrtf(v[k]) * fr;
      const uint32_t d = max(code_of(r, u & 0xfffffu, near), r > 0.f ? 1u : 0u);
      cm[k / 4] |= (a | ((__float_as_uint(m[k]) >> 24) & 0x80u)) << (k % 4 * 8);
      cv[k / 4] |= d << (k % 4 * 8);
      u += 2654435761u;
    }
    if (near < 16) {  // one lane in 2000
      u = u0;
#pragma unroll
      for (int k = 0; k < 4; ++k) cm[k] = cv[k] = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t a = no_m ? 0u : exact_code(fabsf(m[k]), step_m, fm, u >> 12);
        const float r = sqrtf(v[k]);
        const uint32_t d = no_r ? 0u : max(exact_code(r, step_r, fr, u & 0xfffffu), r > 0.f ? 1u : 0u);
        cm[k / 4] |= (a | ((__float_as_uint(m[k]) >> 24) & 0x80u)) << (k % 4 * 8);
        cv[k / 4] |= d << (k % 4 * 8);
        u += 2654435761u;
      }
    }
    if constexpr (WIDE) {
      st16((uint8_t*)x.m + i, make_uint4(cm[0], cm[1], cm[2], cm[3]));
      st16((uint8_t*)x.v + i, make_uint4(cv[0], cv[1], cv[2], cv[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (i + k < n) {
          ((uint8_t*)x.m)[i + k] = (uint8_t)(cm[k / 4] >> (k % 4 * 8));
          ((uint8_t*)x.v)[i + k] = (uint8_t)(cv[k / 4] >> (k % 4 * 8));
        }
    }
  }
}

template <typename T, int BITS, bool MASTER>
__global__ __launch_bounds__(256) void adamw_kernel(Table table, Betas b, const float* grad_scale) {
  int at = 0;  // the last tensor that begins at or before this workgroup
  for (int s = 32; s > 0; s >>= 1)
    if (at + s < table.count && table.begin[at + s] <= (int)blockIdx.x) at += s;
  const Tensor& x = table.t[at];
  const int64_t i = (int64_t)((int)blockIdx.x - table.begin[at]) * kChunk + threadIdx.x * 16, n = x.n;
  const Coefs c = *(const Coefs*)x.coefs;
  const float gs = grad_scale ? *grad_scale : 1.f;
  const uintptr_t all = (uintptr_t)x.p | (uintptr_t)x.g | (uintptr_t)x.m | (uintptr_t)x.v | (uintptr_t)x.master;
  // whole vectors where every pointer allows them and the workgroup is full; its 16 lanes of a block agree either way
  const bool wide = (all & 15) == 0 && (int64_t)((int)blockIdx.x - table.begin[at] + 1) * kChunk <= n;
  if (wide) {
    step_of<T, BITS, MASTER, true>(x, i, n, c, b, gs);
  } else {
    step_of<T, BITS, MASTER, false>(x, i, n, c, b, gs);
  }
}

template <typename T>
void launch(const Table& table, int bits, bool master, unsigned blocks, const Betas& b, const float* gs, hipStream_t st) {
  if (bits == 32) {
    if (master)
      hipLaunchKernelGGL((adamw_kernel<T, 32, true>), dim3(blocks), dim3(256), 0, st, table, b, gs);
    else
      hipLaunchKernelGGL((adamw_kernel<T, 32, false>), dim3(blocks), dim3(256), 0, st, table, b, gs);
  } else {
    if (master)
      hipLaunchKernelGGL((adamw_kernel<T, 8, true>), dim3(blocks), dim3(256), 0, st, table, b, gs);
    else
      hipLaunchKernelGGL((adamw_kernel<T, 8, false>), dim3(blocks), dim3(256), 0, st, table, b, gs);
  }
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
    PKM_REQUIRE(t.numel < (1ll << 35), PKM_ERR_UNSUPPORTED, "pkm_adamw_step: tensor %lld has %lld numbers (fewer than 2^35 are supported)",
                (long long)i, (long long)t.numel);
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
