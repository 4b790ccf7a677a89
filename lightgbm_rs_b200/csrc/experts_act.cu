// What the gradients of the gated and the linear layers need before their products: the gradient
// of the values that the activation was given, rounded to 16 bits for the tensor cores, and the
// bias's gradient, summed in f32 from the values before that rounding.
//
//   GATED    dgate = dh up act'(gate), dup = dh act(gate)
//   LINEAR   dpre  = dy act'(pre),     dbias[e] = sum of dpre over expert e's rows
//
// One pass over the data, bound by memory. The results go to scratch whose rows start at 16 bytes,
// so that the products' loads can walk them at any width.
#include <algorithm>

#include "experts.cuh"
#include "experts_act.cuh"

namespace lgbm_b200 {
namespace experts {
namespace {

constexpr int kThreads = 256;

// 8 values to `p`; VEC: at 16 bytes and all of them wanted, else the first n.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], bool vec, int n) {
  if (vec) {
    Raw<T, 8>::store(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}

// 2^LOG lanes a row, 8 columns a lane at a time.
template <typename T, int LOG>
__global__ void __launch_bounds__(kThreads)
    k_gated_grad(const T* __restrict__ dh, int64_t dh_pitch, bool dh_vec,
                 const T* __restrict__ pre, int64_t pre_pitch, int act, int64_t rows, int hidden,
                 T* __restrict__ dpre, int64_t dpre_pitch) {
  constexpr int kLanes = 1 << LOG;
  const int lane = threadIdx.x % kLanes;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (r >= rows) return;
  const T* dh_row = dh + r * dh_pitch;
  const T* pre_row = pre + r * 2 * pre_pitch;
  T* out = dpre + r * dpre_pitch;
  const bool up_vec = hidden % 8 == 0;
#pragma unroll 2
  for (int c = lane * 8; c < hidden; c += kLanes * 8) {
    const int n = hidden - c;
    Raw<T, 8> rd, rg, ru;
    rg.load(pre_row + c);
    ru.load(pre_row + pre_pitch + c);
    if (dh_vec && n >= 8) rd.load(dh_row + c);
    else rd.load_some(dh_row + c, n);
    float d[8], g[8], u[8], a[8], s[8];
    rg.get(g);
    ru.get(u);
    rd.get(d);
    activate_both(act, g, a, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = d[i] * u[i] * s[i];
      a[i] = d[i] * a[i];
    }
    store8(out + c, s, n >= 8, n);
    store8(out + hidden + c, a, up_vec, n);
  }
}

// Rows of a block, lanes of a row: what the sums' places follow from.
struct SumShape {
  int lanes;       // of a row, a power of two; 8 columns each
  int64_t slabs;   // blocks along the columns
  int64_t blocks;  // blocks along the rows
  int64_t rows;    // of a block
};
SumShape sum_shape(int64_t rows, int32_t outer) {
  SumShape s;
  s.lanes = 1;
  while (s.lanes < 32 && s.lanes * 8 < outer) s.lanes *= 2;
  s.slabs = (outer + s.lanes * 8 - 1) / (s.lanes * 8);
  // eight blocks an SM, of 32 rows at least, and no more than grid.y takes
  const int64_t want = std::max<int64_t>(1, 148 * 8 / s.slabs);
  s.rows = std::max<int64_t>(32, (rows + want - 1) / want);
  s.blocks = (rows + s.rows - 1) / s.rows;
  return s;
}

// Block (x, y) takes rows y R .. and a slab of columns. Where an expert's rows end inside, its
// sums so far go to place y + e: along the rows one of the two grows at every step, so no two
// pieces share a place, and the joining kernel finds an expert's pieces from its offsets alone.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_linear_grad(const T* __restrict__ dy, int64_t dy_pitch, bool dy_vec,
                  const T* __restrict__ pre, int64_t pre_pitch, int act,
                  const int32_t* __restrict__ offsets, int experts, int64_t rows,
                  int64_t rows_a_block, int outer, int lanes, T* __restrict__ dpre,
                  int64_t dpre_pitch, float* __restrict__ sums) {
  __shared__ float part[kThreads * 8];
  const int lane = threadIdx.x % lanes, sub = threadIdx.x / lanes, subs = kThreads / lanes;
  const int64_t c = ((int64_t)blockIdx.x * lanes + lane) * 8;
  const int n = c < outer ? (int)min((int64_t)8, outer - c) : 0;
  const int64_t begin = (int64_t)blockIdx.y * rows_a_block,
                end = min(rows, begin + rows_a_block);
  int64_t row = begin;
  while (row < end) {
    // the expert of `row`: the first whose rows end behind it. Offsets that decrease give some
    // expert and some end, both inside.
    int64_t stop = end;
    int e = experts;
    if (sums) {
      int lo = 0, hi = experts;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid + 1] > row) hi = mid; else lo = mid + 1;
      }
      e = lo;
      if (e < experts) {
        if (row < offsets[e]) {  // before the first expert's
          stop = min(end, (int64_t)offsets[e]);
          e = experts;
        } else {
          stop = min(end, (int64_t)offsets[e + 1]);
        }
      }
    }
    float acc[8] = {};
    if (n > 0) {
#pragma unroll 4
      for (int64_t r = row + sub; r < stop; r += subs) {
        Raw<T, 8> rd, rp;
        if (dy_vec && n == 8) rd.load(dy + r * dy_pitch + c);
        else rd.load_some(dy + r * dy_pitch + c, n);
        float d[8];
        if (pre) {
          rp.load(pre + r * pre_pitch + c);
          float v[8], a[8], s[8];
          rp.get(v);
          rd.get(d);
          activate_both(act, v, a, s);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] *= s[i];
          store8(dpre + r * dpre_pitch + c, d, n == 8, n);
        } else {
          rd.get(d);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += d[i];
      }
    }
    if (e < experts) {
      // [sub][8 lanes' columns], added up in sub's order
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) part[sub * lanes * 8 + lane * 8 + i] = acc[i];
      __syncthreads();
      const int64_t c0 = (int64_t)blockIdx.x * lanes * 8;
      for (int j = threadIdx.x; j < lanes * 8; j += kThreads) {
        float s = 0.0f;
        for (int k = 0; k < subs; ++k) s += part[k * lanes * 8 + j];
        if (c0 + j < outer) sums[((int64_t)blockIdx.y + e) * outer + c0 + j] = s;
      }
    }
    row = stop;
  }
}

// dbias[e][n]: the pieces of expert e, from the block of its first row to that of its last, always
// in the same order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_join_bias(const float* __restrict__ sums, const int32_t* __restrict__ offsets, int64_t rows,
                int64_t rows_a_block, int64_t blocks, int outer, T* __restrict__ dbias) {
  __shared__ float part[kThreads];
  const int e = blockIdx.y, j = threadIdx.x % 32, k = threadIdx.x / 32;
  const int64_t n = (int64_t)blockIdx.x * 32 + j;
  const int64_t lo = min(max((int64_t)offsets[e], (int64_t)0), rows),
                hi = min(max((int64_t)offsets[e + 1], (int64_t)0), rows);
  float s = 0.0f;
  if (n < outer && hi > lo) {
    const int64_t last = min((hi - 1) / rows_a_block, blocks - 1);
    for (int64_t b = lo / rows_a_block + k; b <= last; b += kThreads / 32)
      s += sums[(b + e) * outer + n];
  }
  part[threadIdx.x] = s;
  __syncthreads();
  if (k == 0 && n < outer) {
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) s += part[i * 32 + j];
    dbias[(int64_t)e * outer + n] = from_f32<T>(s);
  }
}

template <typename T>
cudaError_t gated_grad(const void* dh, int64_t dh_pitch, const void* pre, int32_t act, int64_t rows,
                       int32_t hidden, void* dpre, int64_t dpre_pitch, cudaStream_t st) {
  const bool vec = aligned16(dh) && dh_pitch % 8 == 0;
  auto go = [&](auto log) {
    constexpr int kRows = kThreads >> decltype(log)::value;
    const int64_t blocks = (rows + kRows - 1) / kRows;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    k_gated_grad<T, decltype(log)::value><<<(unsigned)blocks, kThreads, 0, st>>>(
        static_cast<const T*>(dh), dh_pitch, vec, static_cast<const T*>(pre), pre_pitch(hidden),
        act, rows, hidden, static_cast<T*>(dpre), dpre_pitch);
    return cudaGetLastError();
  };
  if (hidden <= 16) return go(std::integral_constant<int, 1>());
  if (hidden <= 64) return go(std::integral_constant<int, 3>());
  if (hidden <= 128) return go(std::integral_constant<int, 4>());
  return go(std::integral_constant<int, 5>());
}

template <typename T>
cudaError_t linear_grad(const LinearGrad& c, cudaStream_t st) {
  const SumShape s = sum_shape(c.rows, c.outer);
  const bool vec = aligned16(c.dy) && c.dy_pitch % 8 == 0;
  const dim3 grid((unsigned)s.slabs, (unsigned)s.blocks);
  k_linear_grad<T><<<grid, kThreads, 0, st>>>(
      static_cast<const T*>(c.dy), c.dy_pitch, vec,
      c.dpre ? static_cast<const T*>(c.pre) : nullptr, pre_pitch(c.outer), c.act, c.offsets,
      c.experts, c.rows, s.rows, c.outer, s.lanes, static_cast<T*>(c.dpre), c.dpre_pitch,
      c.dbias ? c.sums : nullptr);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess || !c.dbias) return err;
  const dim3 joins((unsigned)((c.outer + 31) / 32), (unsigned)c.experts);
  if (c.grad_dtype == LGBM_B200_DTYPE_F32)
    k_join_bias<float><<<joins, kThreads, 0, st>>>(c.sums, c.offsets, c.rows, s.rows, s.blocks,
                                                   c.outer, static_cast<float*>(c.dbias));
  else
    k_join_bias<T><<<joins, kThreads, 0, st>>>(c.sums, c.offsets, c.rows, s.rows, s.blocks,
                                               c.outer, static_cast<T*>(c.dbias));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gated_grad(const void* dh, int64_t dh_pitch, const void* pre, int32_t dtype,
                              int32_t act, int64_t rows, int32_t hidden, void* dpre,
                              int64_t dpre_pitch, cudaStream_t st) {
  return dtype == LGBM_B200_DTYPE_BF16
             ? gated_grad<__nv_bfloat16>(dh, dh_pitch, pre, act, rows, hidden, dpre, dpre_pitch, st)
             : gated_grad<__half>(dh, dh_pitch, pre, act, rows, hidden, dpre, dpre_pitch, st);
}

int64_t linear_grad_workspace(int64_t rows, int32_t experts, int32_t outer) {
  if (rows < 1) return 0;
  return (int64_t)sizeof(float) * (sum_shape(rows, outer).blocks + experts) * outer;
}

cudaError_t launch_linear_grad(const LinearGrad& c, cudaStream_t st) {
  return c.dtype == LGBM_B200_DTYPE_BF16 ? linear_grad<__nv_bfloat16>(c, st)
                                         : linear_grad<__half>(c, st);
}

}  // namespace experts
}  // namespace lgbm_b200
