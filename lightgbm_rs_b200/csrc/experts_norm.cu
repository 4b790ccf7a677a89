// The norm of all gradients of a training step, and the gradients scaled to a largest norm.
//
//   norm = sqrt(sum over tensors and elements of g^2),   out = g min(1, max_norm / norm)
//
// Tensors of any number, size, type and alignment in one launch: a table of them is a kernel
// argument (1024 a launch), which the first kernel leaves in memory for the second (30 KB of
// arguments cost the host 7 us a launch). Each is cut into windows of 32 KB of memory that start at
// 16 bytes; a block takes an equal share of all windows, one behind the other, so that one large
// tensor and a thousand small ones are the same work. A thread has 8 loads of 16 bytes in flight.
// The scaling kernel sums the blocks' partial sums itself (592 a launch of 1024 tensors) and walks
// each block's windows from the last to the first: what the first pass read last is still in L2.
//
// Sums. 32 or 64 squares of a thread in f32, then f64. A thread whose f32 sum left the range where
// that is safe (squares overflow from 1.8e19 on, those below 1e-22 lose digits) takes its values
// again in f64, so the norm is right wherever f32 can hold it. Blocks' sums are added in one
// order: the same tensors give the same bits.
//
// Measured, clipped into other memory: 201 million f32 values in 12 tensors 392 us, of which the
// sum is 119 (6.8 TB/s) and the scaling 267 (6.0); 60 million of three types in 1021 tensors 75,
// 28 and 43 (a quarter of the windows are a tensor's ends); 150001 in 5 tensors 6.3, the launch and
// three latencies. Tried without gain: a window ahead in registers (half the blocks an SM), 5 and
// 6 blocks an SM, each window's pieces tested one by one.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "experts.cuh"

namespace lgbm_b200 {
namespace experts {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kPieces = 8;                               // of 16 bytes a thread and window
constexpr int kWindow = kThreads * kPieces * 16;         // bytes
constexpr int kGrid = 4 * 148;                           // blocks of a launch at most
constexpr int kItems = 1024, kFewItems = 64;             // tensors of a launch

template <int ITEMS>
struct Table {
  const char* in[ITEMS];
  char* out[ITEMS];
  int64_t bytes[ITEMS];
  int32_t first[ITEMS + 1];  // window
  uint8_t dtype[ITEMS];
  int32_t items;
};

// A tensor of the table as the first kernel leaves it for the second.
struct alignas(16) Entry {
  const char* in;
  char* out;
  int64_t bytes;
  int32_t first;
  int32_t dtype;
};

// 16 bytes at `at` of memory of which [begin, end) is the tensor: zeros outside. Whole elements.
__device__ __noinline__ uint4 edge_piece(const char* at, const char* begin, const char* end) {
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; i += 2)
    if (at + i >= begin && at + i < end)
      w[i / 4] |= (uint32_t)*reinterpret_cast<const uint16_t*>(at + i) << (8 * (i & 2));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __noinline__ void edge_store(uint4 v, char* to, int from, int end) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 16; i += 2)
    if (i >= from && i < end)
      *reinterpret_cast<uint16_t*>(to + i) = (uint16_t)(w[i / 4] >> (8 * (i & 2)));
}

template <typename T>
__device__ __forceinline__ float2 values(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Sum of the squares of 16 bytes in f64.
template <typename T>
__device__ __noinline__ double precise_sum(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      const double f = __uint_as_float(w[i]);
      d = fma(f, f, d);
    } else {
      const float2 f = values<T>(w[i]);
      d = fma((double)f.x, (double)f.x, d);
      d = fma((double)f.y, (double)f.y, d);
    }
  }
  return d;
}

// This thread's N pieces of a window at `at`, THREADS pieces apart, as the tensor [begin, end)
// fills them.
template <int N, int THREADS>
__device__ __forceinline__ void load_pieces(uint4 (&v)[N], const char* at, const char* begin,
                                            const char* end) {
  const char* p = at + threadIdx.x * 16;
  if (at >= begin && at + N * THREADS * 16 <= end) {  // all of it
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = *reinterpret_cast<const uint4*>(p + j * THREADS * 16);
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j, p += THREADS * 16) {
    v[j] = make_uint4(0, 0, 0, 0);
    if (p >= begin && p + 16 <= end) v[j] = *reinterpret_cast<const uint4*>(p);
    else if (p + 16 > begin && p < end) v[j] = edge_piece(p, begin, end);
  }
}

// Sum of the squares of pieces.
template <typename T, int N>
__device__ __forceinline__ double sum_pieces(const uint4 (&v)[N]) {
  float s[2] = {0.0f, 0.0f};
  uint32_t any = 0;  // a bit of some value but its sign
  constexpr uint32_t kMask = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      any |= w[i] & kMask;
      if constexpr (sizeof(T) == 4) {
        const float f = __uint_as_float(w[i]);
        s[i & 1] = fmaf(f, f, s[i & 1]);
      } else {
        const float2 f = values<T>(w[i]);
        s[0] = fmaf(f.x, f.x, s[0]);
        s[1] = fmaf(f.y, f.y, s[1]);
      }
    }
  }
  const float sum = s[0] + s[1];
  if ((sum >= 1e-28f && sum < 1e37f) || any == 0) return sum;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < N; ++j) d += precise_sum<T>(v[j]);
  return d;
}
template <int N>
__device__ __forceinline__ double sum_pieces(const uint4 (&v)[N], int dtype) {
  if (dtype == LGBM_B200_DTYPE_F32) return sum_pieces<float>(v);
  if (dtype == LGBM_B200_DTYPE_BF16) return sum_pieces<__nv_bfloat16>(v);
  return sum_pieces<__half>(v);
}

// Sum over the block, in every thread.
__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) v += shared[i];
  return v;
}

// The tensor that window w belongs to: the last that starts at or before it (of several that
// start there all but the last are empty).
template <int ITEMS>
__device__ __forceinline__ int item_of(const Table<ITEMS>& t, int w) {
  int lo = 0, hi = t.items;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= w) lo = mid; else hi = mid;
  }
  return lo;
}

// First window of block `b`'s share.
__device__ __forceinline__ int share(int windows, int b, int blocks) {
  return (int)((int64_t)windows * b / blocks);
}

template <int ITEMS>
__global__ void __launch_bounds__(kThreads)
    k_sum_squares(const __grid_constant__ Table<ITEMS> t, double* __restrict__ partial,
                  Entry* __restrict__ entries, int32_t* __restrict__ last) {
  __shared__ double shared[kThreads / 32];
  wait_for_stream();
  let_next_start();
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < t.items; i += gridDim.x * kThreads)
    entries[i] = {t.in[i], t.out[i], t.bytes[i], t.first[i], t.dtype[i]};
  const int windows = t.first[t.items];
  const int begin = share(windows, blockIdx.x, gridDim.x),
            end = share(windows, blockIdx.x + 1, gridDim.x);
  double s = 0.0;
  int item = item_of(t, begin);
  for (int w = begin; w < end; ++w) {
    while (w >= t.first[item + 1]) ++item;
    const char* from = t.in[item];
    const char* at = from - (reinterpret_cast<uintptr_t>(from) & 15) +
                     (int64_t)(w - t.first[item]) * kWindow;
    uint4 v[kPieces];
    load_pieces<kPieces, kThreads>(v, at, from, from + t.bytes[item]);
    s += sum_pieces(v, t.dtype[item]);
  }
  s = block_sum(s, shared);
  if (threadIdx.x == 0) {
    partial[blockIdx.x] = s;
    last[blockIdx.x] = item;
  }
}

// sqrt(s) of f64 as f32: the root of a number in [1, 4) and half its exponent. (A root and a
// quotient of f64 are long chains of dependent instructions, and every block waits for one.)
__device__ __forceinline__ float root(double s) {
  if (!(s > 0.0) || s > 1e300) return (float)s;  // 0, NaN, infinity
  int e = ((int)(__double_as_longlong(s) >> 52) - 1023) & ~1;
  const float m = sqrtf((float)__longlong_as_double(__double_as_longlong(s) -
                                                    ((long long)e << 52)));
  return ldexpf(m, e / 2);
}

// Root of the sum of all partial sums, in the first thread.
__device__ __forceinline__ float norm_of(const double* partial, int count, double* shared) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) s += partial[i];
  s = block_sum(s, shared);
  return threadIdx.x == 0 ? root(s) : 0.0f;
}

__global__ void __launch_bounds__(kThreads)
    k_norm(const double* __restrict__ partial, int count, float* __restrict__ norm) {
  __shared__ double shared[kThreads / 32];
  wait_for_stream();
  let_next_start();
  const float n = norm_of(partial, count, shared);
  if (threadIdx.x == 0) *norm = n;
}

// What all values are multiplied by, one after the other: f, and 1 but for factors below f32's
// normal numbers, where f is the power of two at or above the factor and `rest` keeps its digits. (A
// product with f is then off by 2^-150 at most, and rest is at most 1.)
struct Factor {
  float f, rest;
};

// Two products in one instruction, so that the second factor costs none. (27458 f16 values in 32
// tensors, one cluster: 9.25 us as with one factor, by single products 9.48.)
__device__ __forceinline__ float2 times2(float2 x, float f) {
  uint64_t a, b, r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(x.x), "f"(x.y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(b) : "f"(f));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x.x), "=f"(x.y) : "l"(r));
  return x;
}
template <typename T>
__device__ __forceinline__ uint4 scaled(uint4 v, Factor q) {
  const auto times = [&](float2 x) { return times2(times2(x, q.f), q.rest); };
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 x = times(make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])));
      w[i] = __float_as_uint(x.x);
      w[i + 1] = __float_as_uint(x.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = times(values<T>(w[i]));
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 q2 = __floats2bfloat162_rn(x.x, x.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&q2);
      } else {
        const __half2 q2 = __floats2half2_rn(x.x, x.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&q2);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Pieces scaled, to the same places from `out` on (where the tensor's first element goes).
template <typename T, int N, int THREADS>
__device__ __forceinline__ void store_pieces(const uint4 (&v)[N], const char* at, const char* begin,
                                             const char* end, char* out, Factor f) {
  // the two start alike: 16 bytes of one are 16 bytes of the other
  const bool alike =
      ((reinterpret_cast<uintptr_t>(begin) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const char* p = at + (j * THREADS + threadIdx.x) * 16;
    const uint4 q = scaled<T>(v[j], f);
    char* to = out + (p - begin);
    if (alike && p >= begin && p + 16 <= end)
      *reinterpret_cast<uint4*>(to) = q;
    else if (p + 16 > begin && p < end)
      edge_store(q, to, (int)max((int64_t)(begin - p), (int64_t)0),
                 (int)min((int64_t)(end - p), (int64_t)16));
  }
}
template <int N, int THREADS>
__device__ __forceinline__ void store_pieces(const uint4 (&v)[N], const char* at, const char* begin,
                                             const char* end, char* out, Factor f,
                                             int dtype) {
  if (dtype == LGBM_B200_DTYPE_F32)
    store_pieces<float, N, THREADS>(v, at, begin, end, out, f);
  else if (dtype == LGBM_B200_DTYPE_BF16)
    store_pieces<__nv_bfloat16, N, THREADS>(v, at, begin, end, out, f);
  else
    store_pieces<__half, N, THREADS>(v, at, begin, end, out, f);
}

// The factor that takes norm n to max_norm. A norm of 0 is not above any; NaN stays NaN. A finite
// max_norm beyond f32 is below an infinite norm only: 0, not the NaN of two infinities.
__device__ __forceinline__ Factor factor_of(float n, double max_norm) {
  constexpr float kLargest = 3.402823466e38f;
  if (n <= max_norm) return {1.0f, 1.0f};
  if (n > kLargest || !(max_norm < n * 0x1p-126))
    return {__fdiv_rn((float)fmin(max_norm, (double)kLargest), n), 1.0f};
  if (max_norm < 0x1p-150) return {0.0f, 1.0f};  // no result is larger
  // The factor is in [2^-278, 2^-126), max_norm < 4 and n > 2^-24; q, 2^160 times it, is normal.
  const float q = __fdiv_rn((float)(max_norm * 0x1p100), n * 0x1p-60f);
  const int e = max((__float_as_int(q) >> 23) - 127 - 159, -149);
  return {__int_as_float(1 << (e + 149)), q * __int_as_float((-160 - e + 127) << 23)};
}

// Blocks and their windows as in the launch of k_sum_squares that left these entries; last[b] is
// the tensor of block b's last window.
__global__ void __launch_bounds__(kThreads)
    k_scale(const Entry* __restrict__ entries, const int32_t* __restrict__ last, int windows,
            const double* __restrict__ partial, int count, double max_norm,
            float* __restrict__ norm) {
  __shared__ double shared[kThreads / 32];
  __shared__ Factor factor;
  wait_for_stream();
  let_next_start();
  int item = last[blockIdx.x];
  Entry t = entries[item];
  const float n = norm_of(partial, count, shared);
  if (threadIdx.x == 0) {
    if (norm && blockIdx.x == 0) *norm = n;
    factor = factor_of(n, max_norm);
  }
  __syncthreads();
  const Factor f = factor;
  const int begin = share(windows, blockIdx.x, gridDim.x),
            end = share(windows, blockIdx.x + 1, gridDim.x);
  for (int w = end - 1; w >= begin; --w) {
    while (w < t.first) t = entries[--item];
    if (f.f == 1.0f && t.out == t.in) continue;
    const char* at = t.in - (reinterpret_cast<uintptr_t>(t.in) & 15) +
                     (int64_t)(w - t.first) * kWindow;
    uint4 v[kPieces];
    load_pieces<kPieces, kThreads>(v, at, t.in, t.in + t.bytes);
    store_pieces<kPieces, kThreads>(v, at, t.in, t.in + t.bytes, t.out, f, t.dtype);
  }
}

// Few windows: one cluster of up to 8 blocks holds all values in registers, and the sums meet in
// distributed shared memory. One launch, every value read once.
constexpr int kSmallThreads = 512, kSmallBlocks = 8, kSmallEach = 4;
constexpr int kSmallPieces = kWindow / 16 / kSmallThreads;

__global__ void __launch_bounds__(kSmallThreads, 1)
    k_small(const __grid_constant__ Table<kFewItems> t, int scale, double max_norm,
            float* __restrict__ norm) {
  __shared__ double warps[kSmallThreads / 32];
  __shared__ double sum;
  __shared__ Factor factor;
  cg::cluster_group cluster = cg::this_cluster();
  wait_for_stream();
  let_next_start();
  const int windows = t.first[t.items];
  const int begin = share(windows, blockIdx.x, gridDim.x),
            count = share(windows, blockIdx.x + 1, gridDim.x) - begin;
  uint4 v[kSmallEach][kSmallPieces];
  int item[kSmallEach];
  // a window's place in its tensor
  auto place = [&](int w, int i, const char*& at, const char*& from, const char*& to) {
    from = t.in[i];
    at = from - (reinterpret_cast<uintptr_t>(from) & 15) + (int64_t)(w - t.first[i]) * kWindow;
    to = from + t.bytes[i];
  };
#pragma unroll
  for (int k = 0; k < kSmallEach; ++k) {
    item[k] = 0;
    if (k >= count) continue;
    const int i = item[k] = item_of(t, begin + k);
    const char *at, *from, *to;
    place(begin + k, i, at, from, to);
    load_pieces<kSmallPieces, kSmallThreads>(v[k], at, from, to);
  }
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kSmallEach; ++k) {
    if (k < count) s += sum_pieces(v[k], t.dtype[item[k]]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
  if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = threadIdx.x < kSmallThreads / 32 ? warps[threadIdx.x] : 0.0;
#pragma unroll
    for (int d = kSmallThreads / 64; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
    if (threadIdx.x == 0) sum = s;
  }
  cluster.sync();
  if (threadIdx.x < 32) {
    double all = threadIdx.x < gridDim.x ? *cluster.map_shared_rank(&sum, threadIdx.x) : 0.0;
#pragma unroll
    for (int d = kSmallBlocks / 2; d > 0; d >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, d);
    if (threadIdx.x == 0) {
      const float n = root(all);
      if (blockIdx.x == 0) *norm = n;
      factor = factor_of(n, max_norm);
    }
  }
  __syncthreads();
  // this block has read the others' sums; none leaves before all have
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const Factor f = factor;
#pragma unroll
  for (int k = 0; k < kSmallEach; ++k) {
    if (!scale || k >= count) continue;
    const int i = item[k];
    const char *at, *from, *to;
    place(begin + k, i, at, from, to);
    char* out = t.out[i];
    if (f.f == 1.0f && out == from) continue;
    store_pieces<kSmallPieces, kSmallThreads>(v[k], at, from, to, out, f, t.dtype[i]);
  }
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

cudaError_t run_small(const Table<kFewItems>& t, const NormCall& c, cudaStream_t st) {
  const int blocks = std::min(kSmallBlocks, t.first[t.items]);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(kSmallThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see launch_behind
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k_small, t, (int)c.scale, c.max_norm, c.norm);
}

int64_t launches_of(int64_t tensors) { return (tensors + kItems - 1) / kItems; }

// Windows that a tensor reaches into.
int64_t windows_of(const lgbm_b200_experts_tensor& t) {
  const int64_t lead = reinterpret_cast<uintptr_t>(t.in) & 15;
  return t.count == 0 ? 0 : (lead + t.count * elem_size(t.dtype) + kWindow - 1) / kWindow;
}
// Whether one cluster takes all. (Up to 1 MB. Clipped values, one cluster / two launches: 262000 of
// f32 8.3 / 9.4 us; the norm alone 6.2 / 7.0.)
bool is_small(const lgbm_b200_experts_tensor* tensors, int64_t count) {
  int64_t windows = 0;
  for (int64_t i = 0; i < count && i < kFewItems; ++i) windows += windows_of(tensors[i]);
  return count <= kFewItems && windows <= kSmallBlocks * kSmallEach && windows > 0;
}

template <int ITEMS>
cudaError_t run(const NormCall& c, cudaStream_t st) {
  Table<ITEMS> t;
  // the workspace: partial sums of all launches, then the entries and last tensors of each
  const int64_t launches = launches_of(c.count);
  double* const partial = static_cast<double*>(c.workspace);
  Entry* const entries = reinterpret_cast<Entry*>(partial + launches * kGrid);
  int32_t* const last = reinterpret_cast<int32_t*>(entries + launches * kItems);
  int total = 0, launch = 0;
  auto shape = [](int windows) { return std::min(kGrid, windows); };
  auto each = [&](auto&& go, bool fill) {
    launch = 0;
    for (int64_t i = 0; i < c.count;) {
      int items = 0;
      int32_t windows = 0;  // all tensors' fit, the caller checks
      for (; i < c.count && items < ITEMS; ++i) {
        const lgbm_b200_experts_tensor& v = c.tensors[i];
        if (v.count == 0) continue;
        if (fill) {
          t.in[items] = static_cast<const char*>(v.in);
          t.out[items] = static_cast<char*>(v.out);
          t.bytes[items] = v.count * elem_size(v.dtype);
          t.dtype[items] = (uint8_t)v.dtype;
          t.first[items] = windows;
        }
        windows += (int32_t)windows_of(v);
        ++items;
      }
      if (items == 0) continue;
      if (fill) {
        t.items = items;
        t.first[items] = windows;
      }
      const cudaError_t err = go(windows);
      if (err != cudaSuccess) return err;
      ++launch;
    }
    return cudaSuccess;
  };
  if constexpr (ITEMS == kFewItems)
    if (is_small(c.tensors, c.count)) return each([&](int) { return run_small(t, c, st); }, true);
  cudaError_t err = each(
      [&](int windows) {
        const int at = total;
        total += shape(windows);
        return launch_behind(k_sum_squares<ITEMS>, dim3((unsigned)shape(windows)), kThreads, st, t,
                             partial + at, entries + launch * kItems, last + launch * kGrid);
      },
      true);
  if (err != cudaSuccess) return err;
  if (!c.scale || total == 0) {
    return launch_behind(k_norm, dim3(1), kThreads, st, partial, total, c.norm);
  }
  return each(
      [&](int windows) {
        return launch_behind(k_scale, dim3((unsigned)shape(windows)), kThreads, st,
                             entries + launch * kItems, last + launch * kGrid, windows, partial,
                             total, c.max_norm, launch == 0 ? c.norm : nullptr);
      },
      false);
}

}  // namespace

int64_t norm_workspace(const lgbm_b200_experts_tensor* tensors, int64_t count) {
  if (is_small(tensors, count)) return 0;
  return launches_of(count) * (int64_t)(kGrid * (sizeof(double) + sizeof(int32_t)) +
                                          kItems * sizeof(Entry));
}

cudaError_t launch_norm(const NormCall& c, cudaStream_t st) {
  return c.count <= kFewItems ? run<kFewItems>(c, st) : run<kItems>(c, st);
}

}  // namespace experts
}  // namespace lgbm_b200
