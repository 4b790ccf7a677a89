// The norm of all gradients of a training step, and the gradients scaled to a largest norm.
//
//   norm = sqrt(sum over tensors and elements of g^2),   out = g min(1, max_norm / norm)
//
// Tensors of any number, size, type and alignment in one launch: a table of them is a kernel
// argument (1024 a launch), which the first kernel leaves in memory for the second (30 KB of
// arguments cost the host 7 us a launch). Each is cut into windows of 32 KB of memory that start at 16 bytes; a
// block takes an equal share of all windows, one behind the other, so that one large tensor and a
// thousand small ones are the same work. A thread has 8 loads of 16 bytes in flight. The scaling
// kernel sums the blocks' partial sums itself (592 a launch of 1024 tensors) and walks each block's
// windows from the last to the first: what the first pass read last is still in L2.
//
// Sums. 32 or 64 squares of a thread in f32, then f64. A thread whose f32 sum left the range where
// that is safe (squares overflow from 1.8e19 on, those below 1e-22 lose digits) takes its values
// again in f64, so the norm is right wherever f32 can hold it. Blocks' sums are added in one
// order: the same tensors give the same bits.
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
template <typename T>
__device__ __forceinline__ uint4 piece(const char* at, const char* begin, const char* end) {
  if (at >= begin && at + 16 <= end) return *reinterpret_cast<const uint4*>(at);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; i += (int)sizeof(T))
    if (at + i >= begin && at + i < end) {
      if constexpr (sizeof(T) == 4) w[i / 4] = *reinterpret_cast<const uint32_t*>(at + i);
      else w[i / 4] |= (uint32_t)*reinterpret_cast<const uint16_t*>(at + i) << (8 * (i & 2));
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ float2 values(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// This thread's N pieces of memory from `at` on, THREADS pieces apart; `inside`: all are the
// tensor's.
template <typename T, int N, int THREADS>
__device__ __forceinline__ void load_pieces(uint4 (&v)[N], const char* at, const char* begin,
                                            const char* end, bool inside) {
  if (inside) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      v[j] = *reinterpret_cast<const uint4*>(at + (j * THREADS + threadIdx.x) * 16);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      v[j] = piece<T>(at + (j * THREADS + threadIdx.x) * 16, begin, end);
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
  if (sum >= 1e-28f && sum < 1e37f) return sum;
  if (any == 0) return 0.0;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const uint32_t q = i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3];
      if constexpr (sizeof(T) == 4) {
        const double f = __uint_as_float(q);
        d = fma(f, f, d);
      } else {
        const float2 f = values<T>(q);
        d = fma((double)f.x, (double)f.x, d);
        d = fma((double)f.y, (double)f.y, d);
      }
    }
  }
  return d;
}

template <typename T>
__device__ __forceinline__ double window_sum(const char* at, const char* begin, const char* end) {
  uint4 v[kPieces];
  load_pieces<T, kPieces, kThreads>(v, at, begin, end, at >= begin && at + kWindow <= end);
  return sum_pieces<T>(v);
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
    const char* to = from + t.bytes[item];
    if (t.dtype[item] == LGBM_B200_DTYPE_F32) s += window_sum<float>(at, from, to);
    else if (t.dtype[item] == LGBM_B200_DTYPE_BF16) s += window_sum<__nv_bfloat16>(at, from, to);
    else s += window_sum<__half>(at, from, to);
  }
  s = block_sum(s, shared);
  if (threadIdx.x == 0) {
    partial[blockIdx.x] = s;
    last[blockIdx.x] = item;
  }
}

// sqrt of all partial sums, by the whole block.
__device__ __forceinline__ double norm_of(const double* partial, int count, double* shared) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) s += partial[i];
  return sqrt(block_sum(s, shared));
}

__global__ void __launch_bounds__(kThreads)
    k_norm(const double* __restrict__ partial, int count, float* __restrict__ norm) {
  __shared__ double shared[kThreads / 32];
  const double n = norm_of(partial, count, shared);
  if (threadIdx.x == 0) *norm = (float)n;
}

template <typename T>
__device__ __forceinline__ uint4 scaled(uint4 v, float f) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(__uint_as_float(w[i]) * f);
    } else {
      const float2 x = values<T>(w[i]);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 q = __floats2bfloat162_rn(x.x * f, x.y * f);
        w[i] = *reinterpret_cast<const uint32_t*>(&q);
      } else {
        const __half2 q = __floats2half2_rn(x.x * f, x.y * f);
        w[i] = *reinterpret_cast<const uint32_t*>(&q);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Pieces scaled, to the same places from `out` on (where the tensor's first element goes).
template <typename T, int N, int THREADS>
__device__ __forceinline__ void store_pieces(const uint4 (&v)[N], const char* at, const char* begin,
                                             const char* end, bool inside, char* out, float f) {
  // the two start alike: 16 bytes of one are 16 bytes of the other
  const bool alike =
      ((reinterpret_cast<uintptr_t>(begin) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const char* p = at + (j * THREADS + threadIdx.x) * 16;
    const uint4 q = scaled<T>(v[j], f);
    if (alike && (inside || (p >= begin && p + 16 <= end))) {
      *reinterpret_cast<uint4*>(out + (p - begin)) = q;
    } else {
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 16; i += (int)sizeof(T))
        if (p + i >= begin && p + i < end) {
          char* to = out + (p + i - begin);
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(to) = w[i / 4];
          else *reinterpret_cast<uint16_t*>(to) = (uint16_t)(w[i / 4] >> (8 * (i & 2)));
        }
    }
  }
}

template <typename T>
__device__ __forceinline__ void window_scale(const char* at, const char* begin, const char* end,
                                             char* out, float f) {
  uint4 v[kPieces];
  const bool inside = at >= begin && at + kWindow <= end;
  load_pieces<T, kPieces, kThreads>(v, at, begin, end, inside);
  store_pieces<T, kPieces, kThreads>(v, at, begin, end, inside, out, f);
}

// The factor that takes norm n to max_norm. A norm of 0 is not above any; NaN stays NaN.
__device__ __forceinline__ float factor_of(double n, double max_norm) {
  return n <= max_norm ? 1.0f : (float)(max_norm / n);
}

// Blocks and their windows as in the launch of k_sum_squares that left these entries; last[b] is
// the tensor of block b's last window.
__global__ void __launch_bounds__(kThreads)
    k_scale(const Entry* __restrict__ entries, const int32_t* __restrict__ last, int windows,
            const double* __restrict__ partial, int count, double max_norm,
            float* __restrict__ norm) {
  __shared__ double shared[kThreads / 32];
  int item = last[blockIdx.x];
  Entry t = entries[item];
  const double n = norm_of(partial, count, shared);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const float f = factor_of(n, max_norm);
  const int begin = share(windows, blockIdx.x, gridDim.x),
            end = share(windows, blockIdx.x + 1, gridDim.x);
  for (int w = end - 1; w >= begin; --w) {
    while (w < t.first) t = entries[--item];
    if (f == 1.0f && t.out == t.in) continue;
    const char* at = t.in - (reinterpret_cast<uintptr_t>(t.in) & 15) +
                     (int64_t)(w - t.first) * kWindow;
    const char* to = t.in + t.bytes;
    if (t.dtype == LGBM_B200_DTYPE_F32) window_scale<float>(at, t.in, to, t.out, f);
    else if (t.dtype == LGBM_B200_DTYPE_BF16)
      window_scale<__nv_bfloat16>(at, t.in, to, t.out, f);
    else window_scale<__half>(at, t.in, to, t.out, f);
  }
}

// Few windows: one cluster of up to 8 blocks holds all values in registers, and the sums meet in
// distributed shared memory. One launch, every value read once.
constexpr int kSmallThreads = 1024, kSmallBlocks = 8, kSmallEach = 4;
constexpr int kSmallPieces = kWindow / 16 / kSmallThreads;

template <int ITEMS>
__global__ void __launch_bounds__(kSmallThreads, 1)
    k_small(const __grid_constant__ Table<ITEMS> t, int scale, double max_norm,
            float* __restrict__ norm) {
  __shared__ double warps[kSmallThreads / 32];
  __shared__ double sum;
  cg::cluster_group cluster = cg::this_cluster();
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
    return at >= from && at + kWindow <= to;
  };
#pragma unroll
  for (int k = 0; k < kSmallEach; ++k) {
    item[k] = 0;
    if (k >= count) continue;
    const int i = item[k] = item_of(t, begin + k);
    const char *at, *from, *to;
    const bool inside = place(begin + k, i, at, from, to);
    if (t.dtype[i] == LGBM_B200_DTYPE_F32)
      load_pieces<float, kSmallPieces, kSmallThreads>(v[k], at, from, to, inside);
    else
      load_pieces<__half, kSmallPieces, kSmallThreads>(v[k], at, from, to, inside);
  }
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kSmallEach; ++k) {
    if (k >= count) continue;
    const int dtype = t.dtype[item[k]];
    if (dtype == LGBM_B200_DTYPE_F32) s += sum_pieces<float>(v[k]);
    else if (dtype == LGBM_B200_DTYPE_BF16) s += sum_pieces<__nv_bfloat16>(v[k]);
    else s += sum_pieces<__half>(v[k]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
  if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warps[threadIdx.x];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
    if (threadIdx.x == 0) sum = s;
  }
  cluster.sync();
  double n = 0.0;
  for (unsigned r = 0; r < gridDim.x; ++r) n += *cluster.map_shared_rank(&sum, r);
  cluster.sync();  // every block has read this one's sum
  n = sqrt(n);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  if (!scale) return;
  const float f = factor_of(n, max_norm);
#pragma unroll
  for (int k = 0; k < kSmallEach; ++k) {
    if (k >= count) continue;
    const int i = item[k];
    const char *at, *from, *to;
    const bool inside = place(begin + k, i, at, from, to);
    char* out = t.out[i];
    if (f == 1.0f && out == from) continue;
    if (t.dtype[i] == LGBM_B200_DTYPE_F32)
      store_pieces<float, kSmallPieces, kSmallThreads>(v[k], at, from, to, inside, out, f);
    else if (t.dtype[i] == LGBM_B200_DTYPE_BF16)
      store_pieces<__nv_bfloat16, kSmallPieces, kSmallThreads>(v[k], at, from, to, inside, out, f);
    else
      store_pieces<__half, kSmallPieces, kSmallThreads>(v[k], at, from, to, inside, out, f);
  }
}

template <int ITEMS>
void run_small(const Table<ITEMS>& t, const NormCall& c, cudaStream_t st) {
  const int blocks = std::min(kSmallBlocks, t.first[t.items]);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(kSmallThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, k_small<ITEMS>, t, (int)c.scale, c.max_norm, c.norm);
}

int64_t launches_of(int64_t tensors) { return (tensors + kItems - 1) / kItems; }

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
        const int64_t lead = reinterpret_cast<uintptr_t>(v.in) & 15;
        const int64_t bytes = v.count * elem_size(v.dtype);
        if (fill) {
          t.in[items] = static_cast<const char*>(v.in);
          t.out[items] = static_cast<char*>(v.out);
          t.bytes[items] = bytes;
          t.dtype[items] = (uint8_t)v.dtype;
          t.first[items] = windows;
        }
        windows += (int32_t)((lead + bytes + kWindow - 1) / kWindow);
        ++items;
      }
      if (items == 0) continue;
      if (fill) {
        t.items = items;
        t.first[items] = windows;
      }
      go(windows, i == c.count);
      const cudaError_t err = cudaGetLastError();
      if (err != cudaSuccess) return err;
      ++launch;
    }
    return cudaSuccess;
  };
  bool small = false;  // one launch does it all
  cudaError_t err = each(
      [&](int windows, bool end) {
        small = end && launch == 0 && windows <= kSmallBlocks * kSmallEach;
        if (small) {
          run_small(t, c, st);
          return;
        }
        k_sum_squares<ITEMS><<<shape(windows), kThreads, 0, st>>>(
            t, partial + total, entries + launch * kItems, last + launch * kGrid);
        total += shape(windows);
      },
      true);
  if (err != cudaSuccess || small) return err;
  if (!c.scale || total == 0) {
    k_norm<<<1, kThreads, 0, st>>>(partial, total, c.norm);
    return cudaGetLastError();
  }
  return each(
      [&](int windows, bool) {
        k_scale<<<shape(windows), kThreads, 0, st>>>(entries + launch * kItems,
                                                     last + launch * kGrid, windows, partial,
                                                     total, c.max_norm, launch == 0 ? c.norm : nullptr);
      },
      false);
}

}  // namespace

int64_t norm_workspace(int64_t tensors) {
  return launches_of(tensors) * (int64_t)(kGrid * (sizeof(double) + sizeof(int32_t)) +
                                          kItems * sizeof(Entry));
}

cudaError_t launch_norm(const NormCall& c, cudaStream_t st) {
  return c.count <= kFewItems ? run<kFewItems>(c, st) : run<kItems>(c, st);
}

}  // namespace experts
}  // namespace lgbm_b200
