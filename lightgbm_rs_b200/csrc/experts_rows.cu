// Row operators of the expert layer: the weighted combination of each token's rows with its
// gradient, and dropout from a counter-based generator.
#include "experts.cuh"
#include "philox.h"

namespace lgbm_b200 {
namespace experts {
namespace {

constexpr int kRowThreads = 256;

// out[t] = sum_j w[t, j] y[position[t, j]] in f32, rounded once. A row of `lanes` threads a
// token; JC rows are read at a time, all loads before the first use. Bound by memory: 16384
// tokens of 4 rows of 2048 bf16 in 65 us, 336 MB at 5.2 TB/s (rows in random order).
template <typename T, int V, int JC>
__global__ void __launch_bounds__(kRowThreads)
    k_combine(const T* y, int64_t rows, int width, int64_t pitch, const int32_t* position,
              const float* weights, int64_t tokens, int k, int lanes, T* out) {
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / lanes) + threadIdx.x / lanes;
  if (t >= tokens) return;
  for (int c = (threadIdx.x % lanes) * V; c < width; c += lanes * V) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += JC) {
      float w[JC];
      Raw<T, V> v[JC];
      bool in[JC];
#pragma unroll
      for (int j = 0; j < JC; ++j) {
        const int32_t at = j0 + j < k ? position[t * k + j0 + j] : -1;
        in[j] = at >= 0 && at < rows;
        w[j] = weights && j0 + j < k ? weights[t * k + j0 + j] : 1.0f;
        if (in[j]) v[j].load(y + at * pitch + c);
      }
#pragma unroll
      for (int j = 0; j < JC; ++j)
        if (in[j]) {
          float e[V];
          v[j].get(e);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = fmaf(w[j], e[i], acc[i]);
        }
    }
    Raw<T, V>::store(out + t * width + c, acc);
  }
}

// dy[position[t, j]] = w[t, j] dout[t] and dw[t, j] = <dout[t], y[position[t, j]]>, JC chosen
// rows at a time: dout is read once for them. The dot products are summed over the token's
// lanes in a fixed order, so they do not change from run to run. LANES: a warp a token, or a
// block a token where that many warps would leave SMs idle (fewer than 16 an SM): with a
// barrier a token the block took 168 us on 16384 x 4 x 2048 bf16, the warp takes 96 (604 MB at
// 6.3 TB/s).
template <typename T, int V, int LANES, int JC>
__global__ void __launch_bounds__(kRowThreads)
    k_combine_backward(const T* dout, const T* y, int64_t rows, int width, int64_t dout_pitch,
                       int64_t pitch, const int32_t* position, const float* weights,
                       int64_t tokens, int k, T* dy, float* dweights) {
  __shared__ float part[kRowThreads / 32][JC];
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / LANES) + threadIdx.x / LANES;
  const int lane = threadIdx.x % LANES;
  if (t >= tokens) return;  // whole warps: LANES is 32 or the block
  for (int j0 = 0; j0 < k; j0 += JC) {
    int64_t at[JC];
    float w[JC], dot[JC];
#pragma unroll
    for (int j = 0; j < JC; ++j) {
      at[j] = -1;
      w[j] = dot[j] = 0.0f;
      if (j0 + j < k) {
        const int32_t p = position[t * k + j0 + j];
        if (p >= 0 && p < rows) at[j] = p;
        w[j] = weights ? weights[t * k + j0 + j] : 1.0f;
      }
    }
    for (int c = lane * V; c < width; c += LANES * V) {
      Raw<T, V> rg, rv[JC];
      rg.load(dout + t * dout_pitch + c);
#pragma unroll
      for (int j = 0; j < JC; ++j)
        if (at[j] >= 0 && dweights) rv[j].load(y + at[j] * pitch + c);
      float g[V];
      rg.get(g);
#pragma unroll
      for (int j = 0; j < JC; ++j) {
        if (at[j] < 0) continue;
        float d[V];
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = w[j] * g[i];
        Raw<T, V>::store(dy + at[j] * width + c, d);
        if (dweights) {
          rv[j].get(d);
#pragma unroll
          for (int i = 0; i < V; ++i) dot[j] = fmaf(g[i], d[i], dot[j]);
        }
      }
    }
    if (!dweights) continue;
#pragma unroll
    for (int j = 0; j < JC; ++j)
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], d);
    if constexpr (LANES > 32) {
      if (threadIdx.x % 32 == 0)
#pragma unroll
        for (int j = 0; j < JC; ++j) part[threadIdx.x / 32][j] = dot[j];
      __syncthreads();
      if (threadIdx.x == 0)
#pragma unroll
        for (int j = 0; j < JC; ++j) {
          float s = 0.0f;
          for (int i = 0; i < LANES / 32; ++i) s += part[i][j];
          if (j0 + j < k) dweights[t * k + j0 + j] = s;
        }
      __syncthreads();
    } else if (lane == 0) {
#pragma unroll
      for (int j = 0; j < JC; ++j)
        if (j0 + j < k) dweights[t * k + j0 + j] = dot[j];
    }
  }
}

// Blocks of eight elements a thread. Bound by memory: 32768 x 4096 bf16 take 87 us (537 MB at
// 6.2 TB/s), with a residual 115 (805 MB at 7.0). The generator is about 60 of the 110
// instructions of a block of eight; 32 bits an element instead of 16 would be two generators a
// block and put the instructions above the memory's time.
constexpr int kDropUnroll = 2;

// Element i takes 16 bits of block i / 8 and is kept when they are at least `drop`: the mask
// is recomputed wherever it is needed and never stored. With cut = drop * 2^16 - 1 a high
// half is kept when its whole word is above cut, and a low half when it is after a shift by
// 16: no half is taken out of its word. (drop 2^16 gives the cut 2^32 - 1, which nothing
// passes; drop 0 would need -1 and is a flag.) A dropped element is 0 whatever it held. A
// thread makes kDropUnroll blocks and handles their eight elements each, all loads first.
// VEC: rows of one pitch that 16-byte accesses can walk; a contiguous array is one row.
// FULL: no end of the array inside the block of threads.
template <typename T, bool VEC, bool RES, bool FULL>
__device__ __forceinline__ void drop_block(const T* __restrict__ x, const T* __restrict__ residual,
                                           int64_t n, int64_t width, int64_t pitch,
                                           int64_t residual_pitch, uint32_t cut, bool all,
                                           float scale, uint32_t k0, uint32_t k1,
                                           uint64_t offset, T* __restrict__ out) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  constexpr int kParts = 8 / V;
  const int64_t b0 = (int64_t)blockIdx.x * (kRowThreads * kDropUnroll) + threadIdx.x;
  Raw<T, V> v[kDropUnroll][kParts], a[kDropUnroll][RES ? kParts : 1];
#pragma unroll
  for (int u = 0; u < kDropUnroll; ++u) {
    const int64_t i0 = (b0 + u * kRowThreads) * 8;
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      const int64_t i = i0 + h * V;
      if (FULL || i < n) {
        int64_t at = i, rat = i;
        if (!FULL && width != n) {
          const int64_t r = i / width, c = i - r * width;
          at = r * pitch + c;
          rat = r * residual_pitch + c;
        }
        if (FULL || i + V <= n) {
          v[u][h].load(x + at);
          if constexpr (RES) a[u][h].load(residual + rat);
        } else {
          v[u][h].load_some(x + at, (int)(n - i));
          if constexpr (RES) a[u][h].load_some(residual + rat, (int)(n - i));
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kDropUnroll; ++u) {
    const int64_t b = b0 + u * kRowThreads;
    if (!FULL && b * 8 >= n) break;
    uint32_t words[4];
    philox((uint64_t)b, offset, k0, k1, words);
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      const int64_t at = b * 8 + h * V;
      if (!FULL && at >= n) break;
      float e[V], r[V];
      v[u][h].get(e);
      if constexpr (RES) a[u][h].get(r);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = h * V + i;
        // a low half has zeros below it after the shift: above cut means at least drop * 2^16
        const uint32_t w = (j & 1) ? words[j / 2] : words[j / 2] << 16;
        e[i] = all || w > cut ? e[i] * scale : 0.0f;
        if constexpr (RES) e[i] += r[i];
      }
      if (FULL || at + V <= n) {
        Raw<T, V>::store(out + at, e);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (at + i < n) out[at + i] = from_f32<T>(e[i]);
      }
    }
  }
}

template <typename T, bool VEC, bool RES>
__global__ void __launch_bounds__(kRowThreads)
    k_dropout(const T* __restrict__ x, const T* __restrict__ residual, int64_t n, int64_t width,
              int64_t pitch, int64_t residual_pitch, uint32_t cut, bool all, float scale,
              uint32_t k0, uint32_t k1, uint64_t offset, T* __restrict__ out) {
  const int64_t end = ((int64_t)blockIdx.x + 1) * (kRowThreads * kDropUnroll * 8);
  if (VEC && width == n && end <= n)
    drop_block<T, VEC, RES, VEC>(x, residual, n, width, pitch, residual_pitch, cut, all, scale,
                                 k0, k1, offset, out);
  else
    drop_block<T, VEC, RES, false>(x, residual, n, width, pitch, residual_pitch, cut, all, scale,
                                   k0, k1, offset, out);
}

// Threads that share a token's row: the smallest power of two that covers it, 1 to 256.
int row_lanes(int64_t vectors) {
  int lanes = 1;
  while (lanes < kRowThreads && lanes < vectors) lanes *= 2;
  return lanes;
}

template <typename F>
cudaError_t with_type(int32_t dtype, F&& f) {
  if (dtype == LGBM_B200_DTYPE_F32) return f(float());
  if (dtype == LGBM_B200_DTYPE_BF16) return f(__nv_bfloat16());
  return f(__half());
}

template <typename T, int V>
cudaError_t combine_typed(const T* y, int64_t rows, int width, int64_t pitch,
                          const int32_t* position, const float* weights, int64_t tokens, int k,
                          T* out, cudaStream_t st) {
  const int lanes = row_lanes((width + V - 1) / V);
  const int64_t per_block = kRowThreads / lanes;
  const unsigned blocks = (unsigned)((tokens + per_block - 1) / per_block);
  if (k <= 2)
    k_combine<T, V, 2><<<blocks, kRowThreads, 0, st>>>(y, rows, width, pitch, position, weights,
                                                       tokens, k, lanes, out);
  else
    k_combine<T, V, 4><<<blocks, kRowThreads, 0, st>>>(y, rows, width, pitch, position, weights,
                                                       tokens, k, lanes, out);
  return cudaGetLastError();
}

template <typename T, int V, int LANES>
cudaError_t combine_backward_typed(const T* dout, const T* y, int64_t rows, int width,
                                   int64_t dout_pitch, int64_t pitch, const int32_t* position,
                                   const float* weights, int64_t tokens, int k, T* dy,
                                   float* dweights, cudaStream_t st) {
  const int64_t per_block = kRowThreads / LANES;
  const unsigned blocks = (unsigned)((tokens + per_block - 1) / per_block);
  if (k <= 2)
    k_combine_backward<T, V, LANES, 2><<<blocks, kRowThreads, 0, st>>>(
        dout, y, rows, width, dout_pitch, pitch, position, weights, tokens, k, dy, dweights);
  else
    k_combine_backward<T, V, LANES, 4><<<blocks, kRowThreads, 0, st>>>(
        dout, y, rows, width, dout_pitch, pitch, position, weights, tokens, k, dy, dweights);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_combine(const void* y, int32_t dtype, int64_t rows, int32_t width,
                           int64_t pitch, const int32_t* position, const float* weights,
                           int64_t tokens, int32_t k, void* out, cudaStream_t st) {
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    constexpr int V = 16 / sizeof(T);
    const T* p = static_cast<const T*>(y);
    T* o = static_cast<T*>(out);
    if (width % V == 0 && pitch % V == 0 && aligned16(y) && aligned16(out))
      return combine_typed<T, V>(p, rows, width, pitch, position, weights, tokens, k, o, st);
    return combine_typed<T, 1>(p, rows, width, pitch, position, weights, tokens, k, o, st);
  });
}

cudaError_t launch_combine_backward(const void* dout, const void* y, int32_t dtype,
                                    int64_t rows, int32_t width, int64_t dout_pitch,
                                    int64_t pitch, const int32_t* position,
                                    const float* weights, int64_t tokens, int32_t k, void* dy,
                                    float* dweights, cudaStream_t st) {
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    constexpr int V = 16 / sizeof(T);
    const T* g = static_cast<const T*>(dout);
    const T* p = static_cast<const T*>(y);
    T* o = static_cast<T*>(dy);
    const bool vec = width % V == 0 && dout_pitch % V == 0 && pitch % V == 0 &&
                     aligned16(dout) && aligned16(y) && aligned16(dy);
    auto go = [&](auto v, auto lanes) {
      return combine_backward_typed<T, decltype(v)::value, decltype(lanes)::value>(
          g, p, rows, width, dout_pitch, pitch, position, weights, tokens, k, o, dweights, st);
    };
    using One = std::integral_constant<int, 1>;
    using Vec = std::integral_constant<int, V>;
    using Warp = std::integral_constant<int, 32>;
    using Block = std::integral_constant<int, kRowThreads>;
    const bool wide = tokens < 148 * 16 && (width + (vec ? V : 1) - 1) / (vec ? V : 1) > 64;
    if (vec) return wide ? go(Vec(), Block()) : go(Vec(), Warp());
    return wide ? go(One(), Block()) : go(One(), Warp());
  });
}

cudaError_t launch_dropout(const void* x, const void* residual, int32_t dtype, int64_t rows,
                           int64_t width, int64_t pitch, int64_t residual_pitch, uint32_t drop,
                           uint64_t seed, uint64_t offset, void* out, cudaStream_t st) {
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    constexpr int V = 16 / sizeof(T);
    const int64_t n = rows * width;
    if (n == 0) return cudaSuccess;
    if (pitch == width && (!residual || residual_pitch == width)) {
      width = n;  // contiguous: one row
      pitch = residual_pitch = n;
    }
    // 16 bytes at a time: whole groups of 8 in every row; an array that is one row may end
    // anywhere
    const bool vec = aligned16(x) && aligned16(out) && (!residual || aligned16(residual)) &&
                     (width == n || (width % 8 == 0 && pitch % V == 0 &&
                                     (!residual || residual_pitch % V == 0)));
    const float scale = drop < 65536u ? (float)(65536.0 / (65536.0 - (double)drop)) : 0.0f;
    const uint32_t cut = drop == 0 ? 0u : (uint32_t)(((uint64_t)drop << 16) - 1);
    const int64_t per_block = (int64_t)kRowThreads * kDropUnroll * 8;
    const int64_t want = (n + per_block - 1) / per_block;
    if (want > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    auto go = [&](auto v, auto r) {
      k_dropout<T, decltype(v)::value, decltype(r)::value>
          <<<(unsigned)want, kRowThreads, 0, st>>>(
              static_cast<const T*>(x), static_cast<const T*>(residual), n, width, pitch,
              residual_pitch, cut, drop == 0, scale, (uint32_t)seed, (uint32_t)(seed >> 32),
              offset, static_cast<T*>(out));
    };
    if (vec)
      residual ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
    else
      residual ? go(std::false_type(), std::true_type())
               : go(std::false_type(), std::false_type());
    return cudaGetLastError();
  });
}

}  // namespace experts
}  // namespace lgbm_b200
