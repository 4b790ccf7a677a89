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

// 8 values of 16 bits of a row, loaded first and shifted to their places later. VEC: rows start at
// 16 bytes. Else the aligned pieces that hold them, which may begin before the row and end behind
// it, but not outside of [begin, end), the source.
template <typename T, bool VEC>
struct Eight {
  StagePair v;
  __device__ __forceinline__ void load(const T* p, int n, const T* begin, const T* end) {
    Raw<T, 8> raw;
    if constexpr (VEC) {
      if (n >= 8) raw.load(p);
      else raw.load_some(p, n);
      v.a = raw.bits;
    } else {
      const uintptr_t at = reinterpret_cast<uintptr_t>(p);
      if ((at & ~(uintptr_t)15) >= reinterpret_cast<uintptr_t>(begin) &&
          (at & ~(uintptr_t)15) + 32 <= reinterpret_cast<uintptr_t>(end)) {
        v = stage_load(reinterpret_cast<const char*>(p), 16);
      } else {
        // to where the shift finds them
        raw.load_some(p, n);
        const int s = (int)(at & 15);
        uint32_t w[8] = {raw.bits.x, raw.bits.y, raw.bits.z, raw.bits.w, 0, 0, 0, 0};
#pragma unroll
        for (int i = 7; i > 0; --i)
          w[i] = s & 2 ? __funnelshift_r(w[i - 1], w[i], 16) : w[i];
        w[0] = s & 2 ? w[0] << 16 : w[0];
#pragma unroll
        for (int i = 7; i >= 0; --i) w[i] = s & 4 ? (i >= 1 ? w[i - 1] : 0) : w[i];
#pragma unroll
        for (int i = 7; i >= 0; --i) w[i] = s & 8 ? (i >= 2 ? w[i - 2] : 0) : w[i];
        v.a = make_uint4(w[0], w[1], w[2], w[3]);
        v.b = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
  }
  __device__ __forceinline__ void get(const T* p, float (&f)[8]) const {
    Raw<T, 8> raw;
    if constexpr (VEC) raw.bits = v.a;
    else raw.bits = stage_shift(v, (int)(reinterpret_cast<uintptr_t>(p) & 15), 16);
    raw.get(f);
  }
};

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  __align__(16) T t[8];
  Raw<T, 8>::store(t, v);
  return *reinterpret_cast<const uint4*>(t);
}
// The first n of 8 values.
template <typename T>
__device__ __forceinline__ void store_some(T* p, const float (&v)[8], int n) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = from_f32<T>(v[i]);
}

// 2^LOG lanes a row, 8 columns a lane at a time; blockIdx.y a range of `columns` columns, whole
// steps. ODD: up's columns do not start at 16 bytes. Each lane then writes the 16 bytes that its 8
// columns begin in, of which the first belong to the lane before (a range's first lane finds them
// in a step ahead of it, in which only the last lane works); only where gate ends and up begins
// are values stored one by one. Rows end in padding. Measured: 8192 rows of 2048 in bf16 27 us,
// 6.2 TB/s; 65536 196 us, 6.9; 40009 rows of 129 in f16 24 us, bound by instructions.
template <typename T, int LOG, bool VEC, bool ODD>
__global__ void __launch_bounds__(kThreads)
    k_gated_grad(const T* __restrict__ dh, int64_t dh_pitch, const T* __restrict__ pre,
                 int64_t pre_pitch, int act, int64_t rows, int hidden, int columns,
                 T* __restrict__ dpre, int64_t dpre_pitch) {
  constexpr int kLanes = 1 << LOG;
  wait_for_stream();
  let_next_start();
  const int lane = threadIdx.x % kLanes;
  const int64_t r0 = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  const bool here = r0 < rows;
  const int64_t r = here ? r0 : rows - 1;  // (shuffles want whole warps)
  const T* dh_row = dh + r * dh_pitch;
  const T* pre_row = pre + r * 2 * pre_pitch;
  const T* const dh_end = dh + (rows - 1) * dh_pitch + hidden;
  T* out = dpre + r * dpre_pitch;
  const int shift = hidden % 8;
  uint4 carry = make_uint4(0, 0, 0, 0);
  const int begin = blockIdx.y * columns, end = min(hidden, begin + columns);
#pragma unroll 2
  for (int c0 = ODD && begin > 0 ? begin - kLanes * 8 : begin; c0 < end; c0 += kLanes * 8) {
    const int c = c0 + lane * 8, n = c0 < begin && lane < kLanes - 1 ? 0 : hidden - c;
    const bool mine = here && n > 0 && c0 >= begin;
    Raw<T, 8> rg, ru;
    Eight<T, VEC> rd;
    float d[8], g[8], u[8], a[8], s[8];
    if (n > 0) {
      rg.load(pre_row + c);
      ru.load(pre_row + pre_pitch + c);
      rd.load(dh_row + c, n, dh, dh_end);
      rg.get(g);
      ru.get(u);
      rd.get(dh_row + c, d);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = g[i] = u[i] = 0.0f;
    }
    activate_both(act, g, a, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = d[i] * u[i] * s[i];
      a[i] = d[i] * a[i];
    }
    if (mine) {
      if (!ODD || n >= 8) Raw<T, 8>::store(out + c, s);
      else store_some(out + c, s, n);
    }
    if constexpr (!ODD) {
      if (mine) Raw<T, 8>::store(out + hidden + c, a);
    } else {
      const uint4 w = pack8<T>(a);
      // the lane before's, lane 0 the carry
      const auto from = [&](uint32_t v, uint32_t before) {
        const uint32_t q = __shfl_up_sync(0xFFFFFFFFu, v, 1, kLanes);
        return lane == 0 ? before : q;
      };
      const StagePair both{
          make_uint4(from(w.x, carry.x), from(w.y, carry.y), from(w.z, carry.z),
                     from(w.w, carry.w)),
          w};
      carry = make_uint4(__shfl_sync(0xFFFFFFFFu, w.x, kLanes - 1, kLanes),
                         __shfl_sync(0xFFFFFFFFu, w.y, kLanes - 1, kLanes),
                         __shfl_sync(0xFFFFFFFFu, w.z, kLanes - 1, kLanes),
                         __shfl_sync(0xFFFFFFFFu, w.w, kLanes - 1, kLanes));
      if (mine) {
        T* to = out + hidden + c;
        if (c == 0) {
          store_some(to, a, min(n, 8 - shift));
        } else {
          *reinterpret_cast<uint4*>(to - shift) = stage_shift(both, (8 - shift) * 2, 16);
        }
        if (n <= 8 && n > 8 - shift)  // the rest of the last columns
          *reinterpret_cast<uint4*>(to - shift + 8) =
              stage_shift({w, make_uint4(0, 0, 0, 0)}, (8 - shift) * 2, 16);
      }
    }
  }
}

// Rows of a block, lanes of a row: what the sums' places follow from.
constexpr int kAhead = 4;  // rows that a thread has in flight
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
  s.slabs = ((int64_t)outer + s.lanes * 8 - 1) / (s.lanes * 8);
  // eight blocks an SM, of whole steps, and no more than grid.y takes
  const int64_t want = std::max<int64_t>(1, 148 * 8 / s.slabs);
  const int64_t step = kThreads / s.lanes * kAhead;
  s.rows = ((rows + want - 1) / want + step - 1) / step * step;
  s.blocks = (rows + s.rows - 1) / s.rows;
  return s;
}

// The segment of equal experts that `row` is in: its expert (`experts`: of none) and its end, at
// most `end`. Offsets that decrease give some expert and some end behind `row`, both inside.
struct Segment {
  int expert;
  int64_t stop;
};
__device__ __forceinline__ Segment segment_of(const int32_t* offsets, int experts, int64_t row,
                                              int64_t end) {
  int lo = 0, hi = experts;
  while (lo < hi) {  // the first expert whose rows end behind this one
    const int mid = (lo + hi) >> 1;
    if (__ldg(offsets + mid + 1) > row) hi = mid; else lo = mid + 1;
  }
  if (lo == experts) return {experts, end};
  const int64_t first = __ldg(offsets + lo);
  if (row < first) return {experts, min(end, first)};
  return {lo, min(end, (int64_t)__ldg(offsets + lo + 1))};
}

// Block (x, y) takes rows y R .. and a slab of columns. Where an expert's rows end inside, its
// sums so far go to place y + e: along the rows one of the two grows at every step, so no two
// pieces share a place, and the joining kernel finds an expert's pieces from its offsets alone.
// PRE: through the activation, and dpre is written; else dy is only summed. Measured, launches by
// themselves: 8192 rows of 4096 in bf16 37 us and 6 for the join, 5.4 TB/s; 200003 rows of 64, 255
// experts 27 and 6.
template <typename T, bool VEC, bool PRE>
__global__ void __launch_bounds__(kThreads, 3)
    k_linear_grad(const T* __restrict__ dy, int64_t dy_pitch, const T* __restrict__ pre,
                  int64_t pre_pitch, int act, const int32_t* __restrict__ offsets, int experts,
                  int64_t rows, int64_t rows_a_block, int outer, int lanes, T* __restrict__ dpre,
                  int64_t dpre_pitch, float* __restrict__ sums) {
  __shared__ float part[kThreads / 32][32 * 8];
  wait_for_stream();
  let_next_start();
  const int lane = threadIdx.x % lanes, sub = threadIdx.x / lanes, subs = kThreads / lanes;
  const int64_t c = ((int64_t)blockIdx.x * lanes + lane) * 8;
  const int n = c < outer ? (int)min((int64_t)8, outer - c) : 0;
  const T* const dy_end = dy + (rows - 1) * dy_pitch + outer;
  const int64_t begin = (int64_t)blockIdx.y * rows_a_block,
                end = min(rows, begin + rows_a_block);
  float acc[8] = {};
  // the block's sums of expert e, in one order: lanes of a warp, then its warps
  auto flush = [&](int e) {
    for (int d = 16; d >= lanes; d >>= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], d);
    __syncthreads();
    if (threadIdx.x % 32 < lanes) {
#pragma unroll
      for (int i = 0; i < 8; ++i) part[threadIdx.x / 32][i * lanes + lane] = acc[i];
    }
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.x * lanes * 8 + threadIdx.x;
    if (threadIdx.x < lanes * 8 && col < outer) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k)
        s += part[k][threadIdx.x % 8 * lanes + threadIdx.x / 8];
      sums[((int64_t)blockIdx.y + e) * outer + col] = s;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  };
  // a row's 8 columns, and dpre from them
  struct Row {
    Eight<T, VEC> dy;
    Raw<T, 8> pre;
  };
  auto load = [&](Row& v, int64_t r) {
    v.dy.load(dy + r * dy_pitch + c, n, dy, dy_end);
    if constexpr (PRE) v.pre.load(pre + r * pre_pitch + c);
  };
  auto take = [&](const Row& v, int64_t r) {
    float d[8];
    v.dy.get(dy + r * dy_pitch + c, d);
    if constexpr (PRE) {
      float p[8], a[8], s[8];
      v.pre.get(p);
      activate_both(act, p, a, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] *= s[i];
      Raw<T, 8>::store(dpre + r * dpre_pitch + c, d);  // rows end in padding
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += d[i];
  };
  Segment at{experts, end};
  for (int64_t base = begin; base < end; base += subs * kAhead) {
    const int64_t next = min(end, base + subs * kAhead);
    Row v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (base + k * subs + sub < end && n > 0) load(v[k], base + k * subs + sub);
    if (sums && base == begin) at = segment_of(offsets, experts, begin, end);
    if (at.stop >= next) {  // all of one segment
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (base + k * subs + sub < end && n > 0) take(v[k], base + k * subs + sub);
    }
    for (int64_t row = base; row < next && at.stop <= next;) {
      if (at.stop < next || row > base) {  // segments end inside: each one's rows
        for (int64_t r = row + sub; r < at.stop && n > 0; r += subs) {
          load(v[0], r);
          take(v[0], r);
        }
      }
      if (at.expert < experts) {
        flush(at.expert);
      } else {  // rows of no expert
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
      }
      row = at.stop;
      if (row < end) at = segment_of(offsets, experts, row, end);
      if (row < next && at.stop > next) {  // the one that goes on
        for (int64_t r = row + sub; r < next && n > 0; r += subs) {
          load(v[0], r);
          take(v[0], r);
        }
      }
    }
  }
}

// dbias[e][n]: the pieces of expert e, from the block of its first row to that of its last, always
// in the same order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_join_bias(const float* __restrict__ sums, const int32_t* __restrict__ offsets, int64_t rows,
                int64_t rows_a_block, int64_t blocks, int outer, T* __restrict__ dbias) {
  __shared__ float part[kThreads];
  wait_for_stream();
  let_next_start();
  const int e = blockIdx.y, j = threadIdx.x % 32, k = threadIdx.x / 32;
  const int64_t n = (int64_t)blockIdx.x * 32 + j;
  const int64_t lo = min(max((int64_t)offsets[e], (int64_t)0), rows),
                hi = min(max((int64_t)offsets[e + 1], (int64_t)0), rows);
  float s = 0.0f;
  if (n < outer && hi > lo) {
    const int64_t last = min((hi - 1) / rows_a_block, blocks - 1);
    constexpr int kStep = kThreads / 32, kLoads = 8;  // on their way at a time
    for (int64_t b = lo / rows_a_block + k; b <= last; b += kStep * kLoads) {
      float v[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        v[i] = b + i * kStep <= last ? sums[(b + i * kStep + e) * outer + n] : 0.0f;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) s += v[i];
    }
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
  auto go = [&](auto log, auto vec, auto odd) {
    constexpr int kRows = kThreads >> decltype(log)::value;
    const int64_t blocks = (rows + kRows - 1) / kRows;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    // Few long rows are divided, four steps a block at least, while there are fewer than 8 blocks
    // an SM (1840 rows of 3200: 24 -> 11 us).
    constexpr int kStep = 8 << decltype(log)::value;
    const int64_t steps = (hidden + kStep - 1) / kStep;
    const int64_t ranges = std::max<int64_t>(
        1, std::min<int64_t>({steps / 4, (148 * 8 + blocks - 1) / blocks, 65535}));
    const int64_t columns = (steps + ranges - 1) / ranges * kStep;
    return launch_behind(
        k_gated_grad<T, decltype(log)::value, decltype(vec)::value, decltype(odd)::value>,
        dim3((unsigned)blocks, (unsigned)((hidden + columns - 1) / columns)), kThreads, st,
        static_cast<const T*>(dh), dh_pitch, static_cast<const T*>(pre), pre_pitch(hidden), act,
        rows, hidden, columns, static_cast<T*>(dpre), dpre_pitch);
  };
  auto with_lanes = [&](auto vec, auto odd) {
    if (hidden <= 16) return go(std::integral_constant<int, 1>(), vec, odd);
    if (hidden <= 64) return go(std::integral_constant<int, 3>(), vec, odd);
    if (hidden <= 128) return go(std::integral_constant<int, 4>(), vec, odd);
    return go(std::integral_constant<int, 5>(), vec, odd);
  };
  const bool vec = aligned16(dh) && dh_pitch % 8 == 0;
  if (hidden % 8 == 0)
    return vec ? with_lanes(std::true_type(), std::false_type())
               : with_lanes(std::false_type(), std::false_type());
  return vec ? with_lanes(std::true_type(), std::true_type())
             : with_lanes(std::false_type(), std::true_type());
}

template <typename T>
cudaError_t linear_grad(const LinearGrad& c, cudaStream_t st) {
  const SumShape s = sum_shape(c.rows, c.outer);
  const dim3 grid((unsigned)s.slabs, (unsigned)s.blocks);
  auto go = [&](auto vec, auto through) {
    return launch_behind(
        k_linear_grad<T, decltype(vec)::value, decltype(through)::value>, grid, kThreads, st,
        static_cast<const T*>(c.dy), c.dy_pitch, static_cast<const T*>(c.pre), pre_pitch(c.outer),
        c.act, c.offsets, c.experts, c.rows, s.rows, c.outer, s.lanes, static_cast<T*>(c.dpre),
        c.dpre_pitch, c.dbias ? c.sums : nullptr);
  };
  const std::true_type yes;
  const std::false_type no;
  const cudaError_t err = aligned16(c.dy) && c.dy_pitch % 8 == 0
                              ? (c.dpre ? go(yes, yes) : go(yes, no))
                              : (c.dpre ? go(no, yes) : go(no, no));
  if (err != cudaSuccess || !c.dbias) return err;
  const dim3 joins((unsigned)((c.outer + 31) / 32), (unsigned)c.experts);
  if (c.grad_dtype == LGBM_B200_DTYPE_F32)
    return launch_behind(k_join_bias<float>, joins, kThreads, st, c.sums, c.offsets, c.rows,
                         s.rows, s.blocks, c.outer, static_cast<float*>(c.dbias));
  return launch_behind(k_join_bias<T>, joins, kThreads, st, c.sums, c.offsets, c.rows, s.rows,
                       s.blocks, c.outer, static_cast<T*>(c.dbias));
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
