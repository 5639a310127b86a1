// Token embedding, forward and the gradient of its table, gfx950.
//
//   out_t = T(scale W[id_t])          dW_v = T(scale sum_{t: id_t = v} dout_t), float32 sums
//
// Ids outside [0, rows) read zeros and have no gradient; the padding id reads its row and has no gradient.
//
// The gradient is dense: every row of dW is written once, so writing V D numbers is what bounds a large vocabulary
// with few tokens, and everything else runs beside it or has to be small.
//   1. embed_sort_kernel: sorts, while other workgroups of it fill dW with zeros. Workgroup b of B
//      (a power of two) owns the ids with id mod B = b, so that frequent ids, which lie side by side in a vocabulary, fall to
//      many. It reads all ids twice (they stay in L2): to count its own for each id and wave, and the tokens of the
//      workgroups before it, which is where its part of the sorted list begins; then
//      to place its tokens, each wave its own stretch of them in order. A stable counting sort in one launch, without
//      atomics that decide an order. Rows of dW without a token are zeroed here.
//   2. embed_sum_kernel: the sorted list in chunks of equal length, whatever the ids: a group of lanes sums the rows of a
//      chunk, run by run. A run inside its chunk is written; what a run has in a chunk that it crosses goes to the workspace.
//   3. embed_join_kernel: adds the pieces of the runs that cross chunks, in order.
// The order of every sum is that of the tokens: the same bits on every run.
//
// Measured, 16384 tokens (ids as texts have them) of 151936 x 1024 bf16: forward 15 us, sort beside the zeros 41 to 47 (the sort
// alone 17; with each workgroup a range of ids, whose first holds half of the tokens, 75), sums 20, join 5.
#include "pkm_common.h"

namespace pkm {
namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMaxBucket = 2048;  // ids of a workgroup: a counter for each and wave, 128 KB of LDS

struct EmbedItem {  // a token in the sorted list
  int32_t token, id, begin, end;  // [begin, end): the places of its id
};

// Unit<T, WIDE>: what one lane reads of a row, 16 bytes or one number.
template <typename T, bool WIDE>
struct Unit {
  static constexpr int N = WIDE ? VecTraits<T>::EPV : 1;
  static __device__ __forceinline__ void load(const T* row, int64_t u, float* f) {
    if constexpr (WIDE) {
      VecTraits<T>::unpack(((const uint4*)row)[u], f);
    } else if constexpr (__is_same(T, float)) {
      f[0] = row[u];
    } else if constexpr (__is_same(T, bf16_t)) {
      f[0] = bf16_to_f32(row[u].x);
    } else {
      f[0] = (float)row[u];
    }
  }
  static __device__ __forceinline__ void store(T* row, int64_t u, const float* f) {
    if constexpr (WIDE) {
      st16_nt((uint4*)row + u, VecTraits<T>::pack(f));
    } else if constexpr (__is_same(T, float)) {
      row[u] = f[0];
    } else if constexpr (__is_same(T, bf16_t)) {
      row[u].x = (uint16_t)f32_to_bf16_bits(f[0]);
    } else {
      row[u] = (f16_t)f[0];
    }
  }
};

template <typename I>
__device__ __forceinline__ int64_t id_of(const void* ids, int64_t t) {
  return (int64_t)((const I*)ids)[t];
}

// 2^lg lanes a token, 256 >> lg tokens a workgroup at a time.
template <typename T, bool WIDE, typename I>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* ids, int64_t tokens, const T* __restrict__ w,
                                                        int64_t rows, int64_t stride, int64_t units, int lg, float scale,
                                                        T* __restrict__ out) {
  using U = Unit<T, WIDE>;
  const int lane = threadIdx.x & ((1 << lg) - 1);
  const int64_t dim = units * U::N, per = 256 >> lg;
  for (int64_t t = blockIdx.x * per + (threadIdx.x >> lg); t < tokens; t += gridDim.x * per) {
    const int64_t id = id_of<I>(ids, t);
    const bool there = id >= 0 && id < rows;
    const T* row = w + (there ? id : 0) * stride;
    for (int64_t u = lane; u < units; u += 1 << lg) {
      float f[U::N];
      if (there) {
        U::load(row, u, f);
#pragma unroll
        for (int k = 0; k < U::N; ++k) f[k] *= scale;
      } else {
#pragma unroll
        for (int k = 0; k < U::N; ++k) f[k] = 0.f;
      }
      U::store(out + t * dim, u, f);
    }
  }
}

// An id's place in workgroup b of 2^lg: 0 .. bucket - 1, or -1: an earlier workgroup's, -2: none of them.
__device__ __forceinline__ int place_of(int64_t id, int64_t rows, int64_t padding, int b, int lg) {
  if (id < 0 || id >= rows || id == padding) return -2;
  const int own = (int)id & ((1 << lg) - 1);
  return own == b ? (int)(id >> lg) : own < b ? -1 : -2;
}

template <typename T, bool WIDE, typename I>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(const void* ids, int64_t tokens, int64_t rows,
                                                                  int64_t units, int64_t padding, int bucket,
                                                                  EmbedItem* __restrict__ items, int32_t* n_items,
                                                                  T* __restrict__ dw, int lg_buckets) {
  const int buckets = 1 << lg_buckets, b = blockIdx.x;
  using U = Unit<T, WIDE>;
  if ((int)blockIdx.x >= buckets) {  // zeros for all of dW
    const int64_t bytes = rows * units * U::N * (int64_t)sizeof(T), vectors = bytes / 16;
    const int64_t step = (int64_t)(gridDim.x - buckets) * kSortThreads;
    const int64_t i0 = (int64_t)((int)blockIdx.x - buckets) * kSortThreads + threadIdx.x;
    for (int64_t i = i0; i < vectors; i += step) st16((uint4*)dw + i, make_uint4(0, 0, 0, 0));
    if (i0 < (bytes - 16 * vectors) / (int64_t)sizeof(T)) {
      const float zero[1] = {0.f};
      Unit<T, false>::store(dw, vectors * (16 / (int64_t)sizeof(T)) + i0, zero);
    }
    return;
  }
  extern __shared__ int32_t counts[];  // [waves][bucket], then the places where each wave's next token of an id goes
  __shared__ int32_t sums[kSortWaves], below_sums[kSortWaves];
  int32_t* const begins = counts + kSortWaves * bucket;  // [bucket]
  int32_t* const totals = begins + bucket;               // [bucket]
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int mine = (int)((rows - b + buckets - 1) >> lg_buckets);  // ids b, b + B, ..: there are no more workgroups than rows
  for (int i = tid; i < kSortWaves * bucket; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  // each wave a stretch of the tokens, whole steps of 64
  const int64_t stretch = ((tokens + kSortThreads - 1) / kSortThreads) * 64;
  const int64_t from = min(stretch * wave, tokens), to = min(from + stretch, tokens);
  int32_t below = 0;
  for (int64_t t = from + lane; t < to; t += 64) {
    const int p = place_of(id_of<I>(ids, t), rows, padding, b, lg_buckets);
    if (p >= 0) atomicAdd(&counts[wave * bucket + p], 1);
    below += p == -1;
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) below += __shfl_xor(below, s);
  if (lane == 0) below_sums[wave] = below;
  __syncthreads();
  // of every id: its total and each wave's share before it; the ids' prefix two neighbours a thread
  int32_t total[kMaxBucket / kSortThreads], sum = 0;
#pragma unroll
  for (int k = 0; k < kMaxBucket / kSortThreads; ++k) {
    const int i = tid * (kMaxBucket / kSortThreads) + k;
    total[k] = 0;
    if (i < mine)
      for (int w = 0; w < kSortWaves; ++w) {
        const int32_t c = counts[w * bucket + i];
        counts[w * bucket + i] = total[k];
        total[k] += c;
      }
    sum += total[k];
  }
  int32_t scan = sum;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int32_t other = __shfl_up(scan, s);
    if (lane >= s) scan += other;
  }
  if (lane == 63) sums[wave] = scan;
  __syncthreads();
  int32_t base = scan - sum, all = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < wave) base += sums[w];
    base += below_sums[w];
    all += sums[w] + below_sums[w];
  }
#pragma unroll
  for (int k = 0; k < kMaxBucket / kSortThreads; ++k) {
    const int i = tid * (kMaxBucket / kSortThreads) + k;
    if (i < mine) {
      begins[i] = base;
      totals[i] = total[k];
      for (int w = 0; w < kSortWaves; ++w) counts[w * bucket + i] += base;
    }
    base += total[k];
  }
  if ((int)blockIdx.x == buckets - 1 && tid == 0) *n_items = all;
  __syncthreads();
  for (int64_t t0 = from; t0 < to; t0 += 64) {
    const int64_t t = t0 + lane;
    const int p = t < to ? place_of(id_of<I>(ids, t), rows, padding, b, lg_buckets) : -2;
    uint64_t left = __ballot(p >= 0);
    while (left) {  // one id at a time: its tokens in the lanes' order
      const int id = __builtin_amdgcn_readlane(p, __builtin_ctzll(left));
      const uint64_t same = __ballot(p == id);
      int32_t* const next = &counts[wave * bucket + id];
      const int32_t at = *next;
      if (p == id) {
        const int32_t place = at + __popcll(same & ((1ull << lane) - 1));
        items[place] = EmbedItem{(int32_t)t, (id << lg_buckets) + b, begins[id], begins[id] + totals[id]};
      }
      if (lane == 0) *next = at + __popcll(same);
      left &= ~same;
    }
  }
  if ((int)gridDim.x > buckets) return;
  // rows without a token: a wave each
  const float zero[U::N] = {};
  for (int i = wave; i < mine; i += kSortWaves)
    if (totals[i] == 0)
      for (int64_t u = lane; u < units; u += 64) U::store(dw + (((int64_t)i << lg_buckets) + b) * units * U::N, u, zero);
}

// A group of 2^lg lanes takes a chunk of the sorted list and 2^lg units of its rows.
// parts: [2][chunks][dim] float32: what a run has in a chunk that it crosses, of the run that the chunk begins in and of
// the one that it ends in.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void embed_sum_kernel(const EmbedItem* __restrict__ items, const int32_t* n_items,
                                                        const T* __restrict__ dout, int64_t units, int lg, int slabs,
                                                        int chunk, int64_t chunks, float scale, T* __restrict__ dw,
                                                        float* __restrict__ parts) {
  using U = Unit<T, WIDE>;
  constexpr int N = U::N, FLIGHT = 8;
  const int64_t task = (int64_t)blockIdx.x * (256 >> lg) + (threadIdx.x >> lg);
  const int64_t c = task / slabs, dim = units * N;
  const int64_t u = ((task - c * slabs) << lg) + (threadIdx.x & ((1 << lg) - 1));
  const int64_t n = *n_items, first = c * chunk, last = min(first + chunk, n);
  if (first >= n || u >= units) return;
  float acc[N] = {};
  for (int64_t j = first; j < last; j += FLIGHT) {
    EmbedItem item[FLIGHT];
    float f[FLIGHT][N];
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) item[k] = items[min(j + k, last - 1)];
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) U::load(dout + (int64_t)item[k].token * dim, u, f[k]);
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) {
      if (j + k >= last) break;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += f[k][e];
      const bool run_ends = j + k + 1 == item[k].end;
      if (!run_ends && j + k + 1 < last) continue;
      if (run_ends && item[k].begin >= first) {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] *= scale;
        U::store(dw + (int64_t)item[k].id * dim, u, acc);
      } else {
        float* const to = parts + ((item[k].begin >= first ? chunks : 0) + c) * dim + u * N;
#pragma unroll
        for (int e = 0; e < N; ++e) to[e] = acc[e];
      }
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = 0.f;
    }
  }
}

// The run that chunk c ends in, if it begins there and goes on: its pieces in order. The workgroup's groups of 2^lg lanes
// take equal stretches of them, joined in order through LDS.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void embed_join_kernel(const EmbedItem* __restrict__ items, const int32_t* n_items,
                                                         int64_t units, int lg, int slabs, int chunk, int64_t chunks,
                                                         float scale, T* __restrict__ dw,
                                                         const float* __restrict__ parts) {
  using U = Unit<T, WIDE>;
  constexpr int N = U::N;
  __shared__ float joined[256 * N];
  const int64_t c = blockIdx.x / slabs, dim = units * N;
  const int64_t first = c * chunk, last = first + chunk, n = *n_items;
  if (last >= n) return;
  const EmbedItem item = items[last - 1];
  if (item.begin < first || item.end <= last) return;
  const int64_t pieces = (item.end - 1) / chunk - c;  // in the chunks behind c
  // as many groups as have four pieces each: the join of their sums is one after the other
  const int group = threadIdx.x >> lg, lane = threadIdx.x & ((1 << lg) - 1);
  const int groups = (int)min((int64_t)256 >> lg, (pieces + 3) / 4);
  const int64_t u = ((blockIdx.x - c * slabs) << lg) + lane;
  float acc[N] = {};
  if (u < units && group < groups) {
    if (group == 0) {
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = parts[(chunks + c) * dim + u * N + e];
    }
    const int64_t a = pieces * group / groups, b = pieces * (group + 1) / groups;
#pragma unroll 8
    for (int64_t i = a; i < b; ++i) {
      const float* const from = parts + (c + 1 + i) * dim + u * N;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += from[e];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) joined[threadIdx.x * N + e] = acc[e];
  __syncthreads();
  if (group == 0 && u < units) {
    for (int g = 1; g < groups; ++g)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += joined[((g << lg) + lane) * N + e];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= scale;
    U::store(dw + (int64_t)item.id * dim, u, acc);
  }
}

int log2_lanes(int64_t units, int most) {
  int lg = 0;
  while ((1 << lg) < units && (1 << lg) < most) ++lg;
  return lg;
}

// log2 of the sort's workgroups: 256, one a CU, fewer for fewer rows, more where the counters of 2048 ids need it.
int lg_buckets_of(int64_t rows) {
  int lg = 0;
  while (lg < 8 && (2ll << lg) <= rows) ++lg;
  while (((rows + (1ll << lg) - 1) >> lg) > kMaxBucket) ++lg;
  return lg;
}

// Tokens of a chunk: short ones fill the GPU with few tokens; the pieces of runs that cross them take 8 bytes of workspace for
// each number of a chunk.
int64_t chunk_of(int64_t tokens) { return tokens <= 32768 ? 16 : 64; }

struct EmbedPlan {
  int64_t chunk, chunks, items_at, parts_at, bytes;
};
bool plan_embed(int64_t tokens, int64_t rows, int64_t dim, EmbedPlan* p) {
  if (tokens < 0 || rows < 0 || dim < 1 || tokens >= (1ll << 31) || rows >= (1ll << 31) || dim >= (1ll << 24)) return false;
  p->chunk = chunk_of(tokens);
  p->chunks = (tokens + p->chunk - 1) / p->chunk;
  p->items_at = 256;
  p->parts_at = p->items_at + (tokens * (int64_t)sizeof(EmbedItem) + 255) / 256 * 256;
  p->bytes = p->parts_at + 2 * p->chunks * dim * 4;
  return true;
}

bool wide_rows(const void* a, const void* b, int64_t stride, int64_t dim, int size) {
  return (((uintptr_t)a | (uintptr_t)b) & 15) == 0 && (dim * size) % 16 == 0 && (stride * size) % 16 == 0;
}

template <typename T, bool WIDE, typename I>
void run_fwd(const void* ids, int64_t tokens, const void* w, int64_t rows, int64_t stride, int64_t dim, float scale,
             void* out, hipStream_t st) {
  const int64_t units = dim / Unit<T, WIDE>::N;
  const int lg = log2_lanes(units, 256);
  int64_t blocks = (tokens + (256 >> lg) - 1) / (256 >> lg);
  if (blocks > 256 * 64) blocks = 256 * 64;
  hipLaunchKernelGGL((embed_fwd_kernel<T, WIDE, I>), dim3((unsigned)blocks), dim3(256), 0, st, ids, tokens, (const T*)w,
                     rows, stride, units, lg, scale, (T*)out);
}

template <typename T, bool WIDE, typename I>
int run_bwd(const void* ids, int64_t tokens, const void* dout, int64_t rows, int64_t dim, int64_t padding, float scale,
            void* dw, const EmbedPlan& p, uint8_t* ws, hipStream_t st) {
  const int64_t units = dim / Unit<T, WIDE>::N;
  const int lg_buckets = lg_buckets_of(rows);
  const int64_t buckets = 1ll << lg_buckets, bucket = (rows + buckets - 1) >> lg_buckets;
  int32_t* n_items = (int32_t*)ws;
  EmbedItem* items = (EmbedItem*)(ws + p.items_at);
  float* parts = (float*)(ws + p.parts_at);
  const size_t lds = (kSortWaves + 2) * bucket * 4;
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)embed_sort_kernel<T, WIDE, I>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return pkm_set_error(PKM_ERR_HIP, "pkm_embed_bwd: %s", hipGetErrorString(e));
  }
  // All of dW is filled beside the sort where the rows that are written again are few: 151936 x 1024 bf16 with 16384 tokens
  // 81 us for all kernels, 93 with the sort zeroing the other rows; with 60000 tokens 185 and 156.
  const bool fill = 4 * tokens <= rows && ((uintptr_t)dw & 15) == 0;
  hipLaunchKernelGGL((embed_sort_kernel<T, WIDE, I>), dim3((unsigned)(buckets + (fill ? 256 : 0))), dim3(kSortThreads), lds, st,
                     ids, tokens, rows, units, padding, (int)bucket, items, n_items, (T*)dw, lg_buckets);
  if (tokens > 0) {
    const int lg = log2_lanes(units, 64);
    const int slabs = (int)((units + (1 << lg) - 1) >> lg);
    const int64_t tasks = p.chunks * slabs, per = 256 >> lg;
    hipLaunchKernelGGL((embed_sum_kernel<T, WIDE>), dim3((unsigned)((tasks + per - 1) / per)), dim3(256), 0, st, items,
                       n_items, (const T*)dout, units, lg, slabs, (int)p.chunk, p.chunks, scale, (T*)dw, parts);
    if (p.chunks > 1)
      hipLaunchKernelGGL((embed_join_kernel<T, WIDE>), dim3((unsigned)((p.chunks - 1) * slabs)), dim3(256), 0, st, items,
                         n_items, units, lg, slabs, (int)p.chunk, p.chunks, scale, (T*)dw, parts);
  }
  return pkm_check_launch("pkm_embed_bwd");
}

}  // namespace
}  // namespace pkm

using namespace pkm;

#define EMBED_REQUIRE_COMMON(fn)                                                                                      \
  PKM_REQUIRE(dtype == PKM_DTYPE_F32 || dtype == PKM_DTYPE_BF16 || dtype == PKM_DTYPE_F16, PKM_ERR_INVALID_ARGUMENT,  \
              fn ": dtype %d", dtype);                                                                                \
  PKM_REQUIRE(ids_bits == 32 || ids_bits == 64, PKM_ERR_INVALID_ARGUMENT, fn ": ids of %d bits (32 or 64)", ids_bits); \
  PKM_REQUIRE(tokens >= 0 && rows >= 0 && dim >= 0, PKM_ERR_INVALID_ARGUMENT, fn ": negative size");                  \
  PKM_REQUIRE(tokens < (1ll << 31) && rows < (1ll << 31) && dim < (1ll << 24), PKM_ERR_UNSUPPORTED,                   \
              fn ": %lld tokens, %lld rows of %lld (fewer than 2^31, 2^31 and 2^24 are supported)", (long long)tokens, \
              (long long)rows, (long long)dim)

// f<T, WIDE, I>(...) by dtype, vector width and ids
#define EMBED_DISPATCH(f, ...)                                                                             \
  (dtype == PKM_DTYPE_F32                                                                                  \
       ? (wide ? (ids_bits == 64 ? f<float, true, int64_t>(__VA_ARGS__) : f<float, true, int32_t>(__VA_ARGS__))      \
               : (ids_bits == 64 ? f<float, false, int64_t>(__VA_ARGS__) : f<float, false, int32_t>(__VA_ARGS__)))   \
   : dtype == PKM_DTYPE_BF16                                                                               \
       ? (wide ? (ids_bits == 64 ? f<bf16_t, true, int64_t>(__VA_ARGS__) : f<bf16_t, true, int32_t>(__VA_ARGS__))    \
               : (ids_bits == 64 ? f<bf16_t, false, int64_t>(__VA_ARGS__) : f<bf16_t, false, int32_t>(__VA_ARGS__))) \
       : (wide ? (ids_bits == 64 ? f<f16_t, true, int64_t>(__VA_ARGS__) : f<f16_t, true, int32_t>(__VA_ARGS__))      \
               : (ids_bits == 64 ? f<f16_t, false, int64_t>(__VA_ARGS__) : f<f16_t, false, int32_t>(__VA_ARGS__))))

extern "C" int pkm_embed_fwd(const void* ids, int ids_bits, int64_t tokens, const void* weight, int64_t rows,
                             int64_t row_stride, int64_t dim, int dtype, float scale, void* out, void* stream) {
  EMBED_REQUIRE_COMMON("pkm_embed_fwd");
  if (tokens == 0 || dim == 0) return PKM_OK;
  PKM_REQUIRE(ids && out && (weight || rows == 0), PKM_ERR_INVALID_ARGUMENT, "pkm_embed_fwd: null pointer");
  PKM_REQUIRE(row_stride >= 0 && row_stride < (1ll << 31), PKM_ERR_INVALID_ARGUMENT, "pkm_embed_fwd: row stride %lld",
              (long long)row_stride);
  const bool wide = wide_rows(weight, out, row_stride, dim, elem_size(dtype));
  EMBED_DISPATCH(run_fwd, ids, tokens, weight, rows, row_stride, dim, scale, out, (hipStream_t)stream);
  return pkm_check_launch("pkm_embed_fwd");
}

extern "C" size_t pkm_embed_bwd_workspace_size(int64_t tokens, int64_t rows, int64_t dim) {
  EmbedPlan p;
  return plan_embed(tokens, rows, dim, &p) ? (size_t)p.bytes : 0;
}

extern "C" int pkm_embed_bwd(const void* ids, int ids_bits, int64_t tokens, const void* grad_out, int64_t rows, int64_t dim,
                             int dtype, int64_t padding, float scale, void* grad_weight, void* workspace,
                             size_t workspace_bytes, void* stream) {
  EMBED_REQUIRE_COMMON("pkm_embed_bwd");
  if (rows == 0 || dim == 0) return PKM_OK;
  EmbedPlan p;
  plan_embed(tokens, rows, dim, &p);
  PKM_REQUIRE(p.chunks * ((dim + 63) / 64) < (1ll << 24), PKM_ERR_UNSUPPORTED,
              "pkm_embed_bwd: %lld tokens of %lld numbers are too many for one launch", (long long)tokens, (long long)dim);
  PKM_REQUIRE(grad_weight && (tokens == 0 || (ids && grad_out)), PKM_ERR_INVALID_ARGUMENT, "pkm_embed_bwd: null pointer");
  PKM_REQUIRE(workspace_bytes >= (size_t)p.bytes && workspace, PKM_ERR_WORKSPACE,
              "pkm_embed_bwd: workspace of %zu bytes, %lld needed", workspace_bytes, (long long)p.bytes);
  PKM_REQUIRE(((uintptr_t)workspace & 15) == 0, PKM_ERR_INVALID_ARGUMENT, "pkm_embed_bwd: workspace not 16-byte aligned");
  const bool wide = wide_rows(grad_out, grad_weight, dim, dim, elem_size(dtype));
  return EMBED_DISPATCH(run_bwd, ids, tokens, grad_out, rows, dim, padding, scale, grad_weight, p, (uint8_t*)workspace,
                        (hipStream_t)stream);
}
