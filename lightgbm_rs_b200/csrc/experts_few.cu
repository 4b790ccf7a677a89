// Products grouped by expert for a few rows an expert, as in serving: weights of 16 bits, or
// of 4 bits with group scales.
//
//   y[r, n] = sum_k x[r, k] w[e(r), n, k],   4 bits: w = s[e, n, k / G] (q - z)
//
// The time is the weights' way from memory, so every weight is read once and meets all rows
// of its expert (32 at a time) while it is there. A block of 8 warps takes 128 outputs, 16 a
// warp. A warp streams its 16 weight rows through its own ring of asynchronous copies,
// without waiting for other warps, and multiplies with m16n8k16 matrix instructions:
// weights are the 16 rows, tokens the 8 columns. (A 128-row tcgen05 tile would be nearly
// empty, and neither comes near its rate here: a warp multiplies 1 KB of weights in the time
// in which an SM's share of the memory bandwidth delivers it several times over.) A long
// inner axis is split over the blocks of a cluster when there are few outputs, and the
// partial sums meet in distributed shared memory, added in the blocks' order.
//
// 4 bits: two weights a byte, the even one in the low half, so nibble i and i + 4 of a word
// become a pair of 16-bit numbers with one mask and one subtraction: q | magic is exactly
// magic + q (1024 + q in f16, 128 + q in bf16), and minus (magic + z) it is exactly q - z.
// The tokens are staged in that pair order, which a sum over k does not see. Products of
// q - z are summed in f32 inside a scale group and the group's sum is multiplied by its
// scale in f32: no weight is ever rounded.
#include <algorithm>
#include <mutex>

#include <cooperative_groups.h>

#include "experts.cuh"

namespace lgbm_b200 {
namespace experts {
namespace {

namespace cg = cooperative_groups;

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kOutBlock = 16 * kFewWarps;  // outputs of a block
constexpr int kRowBytes = 128;             // of a weight row in a stage
constexpr int kRowPitch = kRowBytes + 16;  // 36 words: 8 rows x 16 bytes hit all banks once
constexpr int kStageBytes = 16 * kRowPitch;
constexpr int kMaxSplit = 8;               // blocks of a cluster

struct FewArgs {
  const void* x;
  int64_t x_rows, x_pitch;
  const int32_t* index;
  const void* w;           // 16 bits: [E][outer][inner]; 4 bits: [E][outer][w_pitch] bytes
  int64_t w_pitch;         // bytes of a weight row
  const void* scales;      // [E][outer][groups], type of x
  const uint8_t* zeros;    // [E][outer][groups] or null: 8
  int32_t group_shift;     // log2 of the group size
  int32_t groups;
  const int32_t* offsets;
  int32_t experts, inner, outer;
  int64_t rows;
  void* y;
  int32_t blocks;          // blocks along the outputs
  int32_t split;           // blocks of a cluster along the inner axis
  int32_t slice;           // inner length of each, a multiple of 256
  int32_t panel;           // inner length of x and scales staged at a time, same
  int32_t x_vec;           // x may be read 16 bytes at a time
  int32_t w_align;         // 16, 8, 4 or 2: alignment of every weight row
};

__device__ __forceinline__ uint32_t shared_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// 16 bytes of global memory to shared, of which the first `valid` (0..16) are read and the
// rest are zeros; `align` is the alignment of `src`.
__device__ __forceinline__ void copy16(uint32_t dst, const char* src, int valid, int align) {
  if (align == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(valid)
                 : "memory");
  } else if (align == 8) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + i),
                   "l"(valid > i ? src + i : src), "r"(min(max(valid - i, 0), 8))
                   : "memory");
  } else if (align == 4) {
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + i),
                   "l"(valid > i ? src + i : src), "r"(min(max(valid - i, 0), 4))
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      uint32_t v = 0;
      if (valid > i) v = *reinterpret_cast<const uint16_t*>(src + i);
      if (valid > i + 2) v |= (uint32_t)*reinterpret_cast<const uint16_t*>(src + i + 2) << 16;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + i), "r"(v) : "memory");
    }
  }
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                  uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
struct Magic;
template <>
struct Magic<__half> {
  static constexpr uint32_t kBits = 0x6400;  // 1024: the low 10 bits count ones
};
template <>
struct Magic<__nv_bfloat16> {
  static constexpr uint32_t kBits = 0x4300;  // 128: the low 7 bits count ones
};

template <typename T>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t sub2<__half>(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t sub2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Layout of a block's shared memory. TILES column tiles of 8 rows make an item.
template <bool W4, int TILES>
struct FewShape {
  static constexpr int kRows = 8 * TILES;
  // sized so that two blocks share an SM
  static constexpr int kMaxPanel = TILES == 1 ? 1024 : 512;
  static constexpr int kRing = TILES == 1 ? 4 : 3;  // stages a warp
  static constexpr int kStageInner = W4 ? 2 * kRowBytes : kRowBytes / 2;
  // bytes of a staged token: the fragment loads of 8 tokens hit different banks
  static __host__ __device__ int token_pitch(int panel) { return panel * 2 + (W4 ? 64 : 16); }
  // 16-bit scales (and zero points) of an output: an odd number of words, 8 rows hit 8 banks
  static __host__ __device__ int scale_pitch(int panel, int shift) { return (panel >> shift) + 2; }
  static __host__ __device__ int tokens(int panel) {
    const int need = kRows * token_pitch(panel), sums = kRows * kOutBlock * 4;
    return need > sums ? need : sums;  // the partial sums lie over the tokens
  }
  static __host__ __device__ int scales(int panel, int shift) {
    return W4 ? (kOutBlock * scale_pitch(panel, shift) * 2 + 15) / 16 * 16 : 0;
  }
  static __host__ int total(int panel, int shift) {
    return tokens(panel) + 2 * scales(panel, shift) + kFewWarps * kRing * kStageBytes;
  }
};

template <typename T, bool W4, int TILES>
__global__ void __launch_bounds__(kFewThreads, 2) k_grouped_few(const FewArgs g) {
  using S = FewShape<W4, TILES>;
  constexpr int kFewRows = S::kRows, kRing = S::kRing;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int32_t item[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tpitch = S::token_pitch(g.panel), spitch = S::scale_pitch(g.panel, g.group_shift);
  uint8_t* tokens = smem;
  T* scales = reinterpret_cast<T*>(smem + S::tokens(g.panel));
  uint16_t* zeros = reinterpret_cast<uint16_t*>(smem + S::tokens(g.panel) +
                                                S::scales(g.panel, g.group_shift));
  const uint32_t ring = shared_addr(smem + S::tokens(g.panel) +
                                    2 * S::scales(g.panel, g.group_shift)) +
                        warp * kRing * kStageBytes;
  const int gq = lane >> 2, tq = lane & 3;  // row and column quad of the matrix fragments

  // The item of this block: rows [begin, begin + n) of one expert. Items are numbered expert
  // by expert, then the rows past the last offset (expert = experts: zeros).
  if (warp == 0) {
    int want = blockIdx.x / (g.blocks * g.split);
    bool found = false;
    for (int i0 = 0; i0 <= g.experts && !found; i0 += 32) {
      const int e = i0 + lane;
      int64_t b = 0, n = 0;
      if (e <= g.experts) {
        b = min(max((int64_t)g.offsets[e], (int64_t)0), g.rows);
        const int64_t end =
            e < g.experts ? min(max((int64_t)g.offsets[e + 1], b), g.rows) : g.rows;
        n = end - b;
      }
      const int items = (int)((n + kFewRows - 1) / kFewRows);
      int s = items;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
        if (lane >= d) s += o;
      }
      const int first = s - items;
      if (want >= first && want < s) {
        item[0] = e;
        item[1] = (int32_t)(b + (int64_t)(want - first) * kFewRows);
        item[2] = (int32_t)min(n - (int64_t)(want - first) * kFewRows, (int64_t)kFewRows);
      }
      const int total = __shfl_sync(0xFFFFFFFFu, s, 31);
      found = want < total;
      want -= total;
    }
    if (!found && lane == 0) item[0] = -1;
  }
  __syncthreads();
  const int expert = item[0], begin = item[1], nrows = item[2];
  if (expert < 0) return;  // the whole cluster has the same item
  const int rank = blockIdx.x % g.split;
  const int out0 = blockIdx.x / g.split % g.blocks * kOutBlock;
  const int k_begin = rank * g.slice, k_end = min(g.inner, k_begin + g.slice);
  T* y = static_cast<T*>(g.y);
  if (expert == g.experts) {
    if (rank == 0)
      for (int i = threadIdx.x; i < nrows * kOutBlock; i += kFewThreads) {
        const int r = i / kOutBlock, n = out0 + i % kOutBlock;
        if (n < g.outer) y[(int64_t)(begin + r) * g.outer + n] = from_f32<T>(0.0f);
      }
    return;
  }

  const int tiles = (nrows + 7) / 8;
  const int my_row0 = out0 + warp * 16;
  const char* wbase = static_cast<const char*>(g.w) +
                      ((int64_t)expert * g.outer + my_row0) * g.w_pitch;
  const int row_bytes = W4 ? (int)g.w_pitch : g.inner * 2;
  const int stages = k_end > k_begin ? (k_end - k_begin + S::kStageInner - 1) / S::kStageInner : 0;
  const int byte0 = W4 ? k_begin / 2 : k_begin * 2;
  auto load_stage = [&](int i) {
    if (i < stages) {
      const int at = byte0 + i * kRowBytes + (lane & 7) * 16;
      const uint32_t dst = ring + (i % kRing) * kStageBytes + (lane & 7) * 16;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = (lane >> 3) + 4 * j;
        int valid = min(max(row_bytes - at, 0), 16);
        if (my_row0 + row >= g.outer) valid = 0;
        const char* src = valid ? wbase + (int64_t)row * g.w_pitch + at
                                : static_cast<const char*>(g.w);
        copy16(dst + row * kRowPitch, src, valid, g.w_align);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float acc[TILES][4];
#pragma unroll
  for (int j = 0; j < TILES; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;

#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) load_stage(i);

  const uint16_t* x = static_cast<const uint16_t*>(g.x);
  int kp = g.panel;  // inner position in the panel
  for (int i = 0; i < stages; ++i, kp += S::kStageInner) {
    if (kp == g.panel) {
      kp = 0;
      const int k0 = k_begin + i * S::kStageInner;
      if (i > 0) __syncthreads();
      // tokens of this panel, 8 inner elements a thread; zeros past the rows and the slice
      const int vecs = g.panel / 8;
      for (int r = warp; r < 8 * tiles; r += kFewWarps) {
        int64_t at = -1;
        if (r < nrows) at = g.index ? g.index[begin + r] : begin + r;
        const bool inside = at >= 0 && at < g.x_rows;
        const uint16_t* src = x + (inside ? at : 0) * g.x_pitch;
        for (int c = lane; c < vecs; c += 32) {
          const int k = k0 + c * 8;
          uint32_t v[4] = {0, 0, 0, 0};
          if (inside && k < k_end) {
            if (g.x_vec && k + 8 <= k_end) {
              const uint4 q = __ldg(reinterpret_cast<const uint4*>(src + k));
              v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (k + j < k_end) v[j / 2] |= (uint32_t)src[k + j] << (16 * (j & 1));
            }
          }
          if (W4) {  // pairs (0, 4), (1, 5), (2, 6), (3, 7)
            const uint32_t p0 = __byte_perm(v[0], v[2], 0x5410),
                           p1 = __byte_perm(v[0], v[2], 0x7632),
                           p2 = __byte_perm(v[1], v[3], 0x5410),
                           p3 = __byte_perm(v[1], v[3], 0x7632);
            v[0] = p0, v[1] = p1, v[2] = p2, v[3] = p3;
          }
          *reinterpret_cast<uint4*>(tokens + r * tpitch + c * 16) =
              make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      if (W4) {
        const int bits = 31 - __clz(g.panel >> g.group_shift);
        const int first = k0 >> g.group_shift;
        for (int p = threadIdx.x; p < kOutBlock << bits; p += kFewThreads) {
          const int r = p >> bits, c = p & ((1 << bits) - 1);
          T s = from_f32<T>(0.0f);
          uint32_t z = 8;
          if (out0 + r < g.outer && first + c < g.groups) {
            const int64_t at = ((int64_t)expert * g.outer + out0 + r) * g.groups + first + c;
            s = static_cast<const T*>(g.scales)[at];
            if (g.zeros) z = g.zeros[at] & 15;
          }
          scales[r * spitch + c] = s;
          zeros[r * spitch + c] = (uint16_t)(Magic<T>::kBits + z);
        }
      }
      __syncthreads();
    }
    load_stage(i + kRing - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
    __syncwarp();
    const uint32_t st = ring + (i % kRing) * kStageBytes;
    if constexpr (W4) {
      const uint32_t a_at = st + gq * kRowPitch + tq * 4;
      const uint8_t* b_at = tokens + gq * tpitch + (kp + tq * 8) * 2;
      const int s_at = (warp * 16 + gq) * spitch;
      float part[TILES][4];
#pragma unroll
      for (int j = 0; j < S::kStageInner / 32; ++j) {
        const int lo = s_at + ((kp + j * 32) >> g.group_shift), hi = lo + 8 * spitch;
        if (((j * 32) & ((1 << g.group_shift) - 1)) == 0) {
#pragma unroll
          for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) part[n][q] = 0.0f;
        }
        uint32_t wl, wh;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(wl) : "r"(a_at + j * 16));
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(wh) : "r"(a_at + j * 16 + 8 * kRowPitch));
        const uint32_t zl = g.zeros ? zeros[lo] * 0x10001u : (Magic<T>::kBits + 8) * 0x10001u;
        const uint32_t zh = g.zeros ? zeros[hi] * 0x10001u : (Magic<T>::kBits + 8) * 0x10001u;
        uint32_t pl[4], ph[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          pl[q] = sub2<T>(((wl >> (4 * q)) & 0x000F000Fu) | Magic<T>::kBits * 0x10001u, zl);
          ph[q] = sub2<T>(((wh >> (4 * q)) & 0x000F000Fu) | Magic<T>::kBits * 0x10001u, zh);
        }
        const uint32_t a0[4] = {pl[0], ph[0], pl[1], ph[1]}, a1[4] = {pl[2], ph[2], pl[3], ph[3]};
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
          if (TILES == 1 || n < tiles) {
            const uint4 b = *reinterpret_cast<const uint4*>(b_at + n * 8 * tpitch + j * 64);
            mma_16816<T>(part[n], a0, b.x, b.y);
            mma_16816<T>(part[n], a1, b.z, b.w);
          }
        }
        if (((j * 32 + 32) & ((1 << g.group_shift) - 1)) == 0) {
          const float sl = to_f32<T>(scales[lo]), sh = to_f32<T>(scales[hi]);
#pragma unroll
          for (int n = 0; n < TILES; ++n) {
            acc[n][0] = fmaf(sl, part[n][0], acc[n][0]);
            acc[n][1] = fmaf(sl, part[n][1], acc[n][1]);
            acc[n][2] = fmaf(sh, part[n][2], acc[n][2]);
            acc[n][3] = fmaf(sh, part[n][3], acc[n][3]);
          }
        }
      }
    } else {
      const uint32_t a_at = st + (lane & 15) * kRowPitch + (lane >> 4) * 16;
      const uint8_t* b_at = tokens + gq * tpitch + kp * 2 + tq * 4;
#pragma unroll
      for (int j = 0; j < S::kStageInner / 16; ++j) {
        uint32_t a[4];
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                     : "r"(a_at + j * 32)
                     : "memory");
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
          if (TILES == 1 || n < tiles) {
            const uint8_t* b = b_at + n * 8 * tpitch + j * 32;
            mma_16816<T>(acc[n], a, *reinterpret_cast<const uint32_t*>(b),
                         *reinterpret_cast<const uint32_t*>(b + 16));
          }
        }
      }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // partial sums as [row][output], over the tokens; with a split inner axis the blocks of
  // the cluster each add up and store a share of the rows
  __syncthreads();
  float* sums = reinterpret_cast<float*>(tokens);
#pragma unroll
  for (int n = 0; n < TILES; ++n)
    if (n < tiles) {
      float* at = sums + (n * 8 + 2 * tq) * kOutBlock + warp * 16 + gq;
      at[0] = acc[n][0];
      at[kOutBlock] = acc[n][1];
      at[8] = acc[n][2];
      at[kOutBlock + 8] = acc[n][3];
    }
  if (g.split == 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < nrows * kOutBlock; i += kFewThreads) {
      const int n = out0 + i % kOutBlock;
      if (n < g.outer)
        y[(int64_t)(begin + i / kOutBlock) * g.outer + n] = from_f32<T>(sums[i]);
    }
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = rank * kFewThreads + threadIdx.x; i < nrows * kOutBlock;
       i += g.split * kFewThreads) {
    float s = 0.0f;
    for (int r = 0; r < g.split; ++r) s += cluster.map_shared_rank(sums, r)[i];
    const int n = out0 + i % kOutBlock;
    if (n < g.outer) y[(int64_t)(begin + i / kOutBlock) * g.outer + n] = from_f32<T>(s);
  }
  cluster.sync();
}

constexpr int kMaxDevices = 64;
struct FewDevice {
  std::mutex mu;
  uint32_t ready = 0;  // instantiations whose shared memory limit is raised, one bit each
};
FewDevice g_few_devices[kMaxDevices];

template <typename T, bool W4, int TILES>
cudaError_t launch_few_tiles(FewArgs g, cudaStream_t st) {
  using S = FewShape<W4, TILES>;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  {
    FewDevice& d = g_few_devices[dev];
    std::lock_guard<std::mutex> lock(d.mu);
    const uint32_t bit = 1u << (4 * (TILES > 1) + 2 * W4 + std::is_same<T, __half>::value);
    if (!(d.ready & bit)) {
      err = cudaFuncSetAttribute(k_grouped_few<T, W4, TILES>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 S::total(S::kMaxPanel, 5));
      if (err != cudaSuccess) return err;
      d.ready |= bit;
    }
  }
  const int64_t blocks = (g.outer + kOutBlock - 1) / kOutBlock;
  const int64_t items = std::min<int64_t>(g.experts + 1, g.rows) + g.rows / S::kRows;
  // Split the inner axis, in steps of at least 512, while the blocks would not fill the SMs.
  const int64_t busy = blocks * std::min<int64_t>(g.experts, g.rows);
  int split = 1;
  while (split < kMaxSplit && split * 1024 <= g.inner && busy * split < 148) split *= 2;
  const int64_t steps = (g.inner + 255) / 256;
  g.blocks = (int32_t)blocks;
  g.split = split;
  g.slice = (int32_t)((steps + split - 1) / split * 256);
  g.panel = 256;
  while (g.panel < S::kMaxPanel && g.panel < g.slice) g.panel *= 2;
  if (blocks * split * items > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(blocks * split * items), 1, 1);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)S::total(g.panel, g.group_shift);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_grouped_few<T, W4, TILES>, g);
}

template <typename T, bool W4>
cudaError_t launch_few_typed(const FewArgs& g, cudaStream_t st) {
  // Items of 8 rows while few experts can have more: no test for absent column tiles in the
  // inner loop, and the tokens of twice the inner length in shared memory.
  return g.rows <= 4 * (int64_t)g.experts || g.rows <= 8 ? launch_few_tiles<T, W4, 1>(g, st)
                                                         : launch_few_tiles<T, W4, 4>(g, st);
}

}  // namespace

cudaError_t launch_few(const FewCall& c, cudaStream_t st) {
  FewArgs g{};
  g.x = c.x;
  g.x_rows = c.x_rows;
  g.x_pitch = c.x_pitch;
  g.index = c.index;
  g.w = c.w;
  g.offsets = c.offsets;
  g.experts = c.experts;
  g.inner = c.inner;
  g.outer = c.outer;
  g.rows = c.rows;
  g.y = c.y;
  g.x_vec = aligned16(c.x) && c.x_pitch % 8 == 0;
  const bool half = c.dtype == LGBM_B200_DTYPE_F16;
  if (c.group_size == 0) {
    g.w_pitch = (int64_t)c.inner * 2;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(c.w) | (uintptr_t)g.w_pitch;
    g.w_align = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
    return half ? launch_few_typed<__half, false>(g, st)
                : launch_few_typed<__nv_bfloat16, false>(g, st);
  }
  g.w_pitch = (c.inner + 31) / 32 * 16;
  g.w_align = 16;
  g.scales = c.scales;
  g.zeros = c.zeros;
  g.group_shift = c.group_size == 32 ? 5 : c.group_size == 64 ? 6 : 7;
  g.groups = (c.inner + c.group_size - 1) / c.group_size;
  return half ? launch_few_typed<__half, true>(g, st)
              : launch_few_typed<__nv_bfloat16, true>(g, st);
}

}  // namespace experts
}  // namespace lgbm_b200
