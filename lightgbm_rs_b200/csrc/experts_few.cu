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
// Measured (2 rows an expert): 16 bits, 32 experts of 4096 x 2048, 537 MB: 90 to 92 us, 5.9 TB/s,
// memory; 8 experts, 29 us, 4.6 TB/s: 256 blocks are 1.7 an SM. 4 bits, 32 experts of 4096 x
// 2000: groups of 128 41 us (3.3 TB/s), of 64 45, of 32 51; bound by instructions, about 50 for the
// 256 bytes that a warp unpacks and multiplies at a time, 14 of them shifts and masks on the
// integer pipe. One row of 8 x 4096 x 4096, two experts: 10 us, of which launch, the joined
// cluster and the chain offsets - index - tokens are most.
#include <algorithm>
#include <atomic>

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
};

__device__ __forceinline__ uint32_t shared_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// 16 bytes of global memory to shared, of which the first `valid` (0..16) are read and the
// rest are zeros. ALIGN: of `src`, 16, 4 or 2 bytes.
template <int ALIGN>
__device__ __forceinline__ void copy16(uint32_t dst, const char* src, int valid) {
  if constexpr (ALIGN == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(valid)
                 : "memory");
  } else if constexpr (ALIGN == 4) {
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
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                         uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (w & mask) | magic in one instruction: with both constants in registers. As immediates they
// took two, and the kernel is bound by the integer pipe (16 rows of 32 x 4096 x 2000: 55 us
// against 51).
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
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

// The low (h = 0) or high half of a word as f32.
template <typename T>
__device__ __forceinline__ float half_of(uint32_t w, int h);
template <>
__device__ __forceinline__ float half_of<__nv_bfloat16>(uint32_t w, int h) {
  return __uint_as_float(h ? w & 0xFFFF0000u : w << 16);
}
template <>
__device__ __forceinline__ float half_of<__half>(uint32_t w, int h) {
  const __half2 v = *reinterpret_cast<__half2*>(&w);
  return h ? __high2float(v) : __low2float(v);
}

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

// A kernel's variant: TILES column tiles of 8 rows make an item; SHIFT is log2 of the scale
// group's size, 0 with weights of 16 bits, whose rows are aligned to ALIGN bytes.
template <typename T_, int TILES_, int SHIFT_, bool ZEROS_, int ALIGN_>
struct FewShape {
  using T = T_;
  static constexpr int TILES = TILES_, SHIFT = SHIFT_, ALIGN = ALIGN_;
  static constexpr bool W4 = SHIFT > 0, ZEROS = ZEROS_;
  // Blocks that share an SM, and stages of a warp's ring: with 4 bits the arithmetic wants
  // warps, with 16 bits the memory wants bytes in flight (4 x 16 KB a block).
  static constexpr int kBlocks = W4 && TILES == 1 ? 3 : 2;
  static constexpr int kRing = !W4 && TILES == 1 ? 5 : 3;
  static constexpr int kMaxPanel = 512;
  static constexpr int kRows = 8 * TILES;
  static constexpr int kStageInner = W4 ? 2 * kRowBytes : kRowBytes / 2;
  // Scales (and zero points) of a warp's 16 outputs in a stage: two sets, one in use; two
  // lanes bring an output's, kScaleLane each. An output's are kScalePitch apart, so that 8
  // outputs hit different banks.
  static constexpr int kGroups = W4 ? kStageInner >> SHIFT : 2;
  static constexpr int kScalePitch = kGroups + 2;
  static constexpr int kScaleBytes = W4 ? 16 * kScalePitch * 2 : 0;
  static constexpr int kScaleLane = kGroups / 2;
  // bytes of a staged token: the fragment loads of 8 tokens hit different banks
  static __host__ __device__ int token_pitch(int panel) { return panel * 2 + (W4 ? 64 : 16); }
  static __host__ __device__ int tokens(int panel) {
    const int need = kRows * token_pitch(panel), sums = kRows * kOutBlock * 4;
    return need > sums ? need : sums;  // the partial sums lie over the tokens
  }
  static __host__ __device__ int ring(int panel) {
    return tokens(panel) + kFewWarps * 2 * (ZEROS ? 2 : 1) * kScaleBytes;
  }
  static __host__ int total(int panel) { return ring(panel) + kFewWarps * kRing * kStageBytes; }
};

template <typename S>
__global__ void __launch_bounds__(kFewThreads, S::kBlocks) k_grouped_few(const FewArgs g) {
  using T = typename S::T;
  constexpr int TILES = S::TILES, SHIFT = S::SHIFT;
  constexpr bool W4 = S::W4;
  constexpr int kFewRows = S::kRows, kRing = S::kRing;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int32_t item[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tpitch = S::token_pitch(g.panel);
  uint8_t* tokens = smem;
  uint8_t* scale_sets =
      smem + S::tokens(g.panel) + warp * 2 * (S::ZEROS ? 2 : 1) * S::kScaleBytes;
  uint8_t* ring = smem + S::ring(g.panel) + warp * kRing * kStageBytes;
  const int gq = lane >> 2, tq = lane & 3;  // row and column quad of the matrix fragments

  // The item of this block: rows [begin, begin + n) of one expert. Items are numbered expert
  // by expert, then the rows past the last offset and those before the first (expert >= experts:
  // zeros).
  if (warp == 0) {
    int want = blockIdx.x / (g.blocks * g.split);
    bool found = false;
    for (int i0 = 0; i0 <= g.experts + 1 && !found; i0 += 32) {
      const int e = i0 + lane;
      int64_t b = 0, n = 0;
      if (e <= g.experts + 1) {
        b = min(max((int64_t)g.offsets[e <= g.experts ? e : 0], (int64_t)0), g.rows);
        const int64_t end =
            e < g.experts ? min(max((int64_t)g.offsets[e + 1], b), g.rows) : g.rows;
        n = end - b;
        if (e > g.experts) n = b, b = 0;
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
  if (expert >= g.experts) {
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
  // this lane's piece of rows lane / 8 + 4 j of a stage
  const char* src0 = wbase + (int64_t)(lane >> 3) * g.w_pitch + byte0 + (lane & 7) * 16;
  const uint32_t dst0 = shared_addr(ring) + (lane >> 3) * kRowPitch + (lane & 7) * 16;
  const int rest0 = row_bytes - byte0 - (lane & 7) * 16, rows_in = g.outer - my_row0 - (lane >> 3);
  const int64_t step4 = 4 * g.w_pitch;
  int load_slot = 0;
  auto load_stage = [&](int i) {
    if (i < stages) {
      const char* src = src0 + i * kRowBytes;  // of the slice's stage i
      const uint32_t dst = dst0 + load_slot * kStageBytes;
      const int rest = rest0 - i * kRowBytes;
      if (S::ALIGN == 16 && my_row0 + 16 <= g.outer &&
          byte0 + (i + 1) * kRowBytes <= row_bytes) {  // all of it exists
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 4 * j * kRowPitch),
                       "l"(src + j * step4)
                       : "memory");
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int valid = 4 * j < rows_in ? min(max(rest, 0), 16) : 0;
          copy16<S::ALIGN>(dst + 4 * j * kRowPitch,
                           valid ? src + j * step4 : static_cast<const char*>(g.w), valid);
        }
      }
    }
    load_slot = load_slot + 1 == kRing ? 0 : load_slot + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // Scales of stage i into registers, and from there into set i % 2: the loads of a stage are
  // in flight while the stage before it is multiplied.
  // (As words, loaded under a branch: a half-register result, or a select behind the load,
  // would wait for it.)
  uint32_t next_scale[S::kScaleLane], next_zero[S::kScaleLane];
  const int scale_row = lane >> 1, scale_col = (lane & 1) * S::kScaleLane;
  const int64_t scale_at = ((int64_t)expert * g.outer + my_row0 + scale_row) * g.groups +
                           (k_begin >> SHIFT) + scale_col;
  const uint16_t* scale_src = static_cast<const uint16_t*>(g.scales) + scale_at;
  const uint8_t* zero_src = S::ZEROS ? g.zeros + scale_at : nullptr;
  // groups left from this lane's first one; none for an output that does not exist
  int scale_left = my_row0 + scale_row < g.outer
                       ? g.groups - (k_begin >> SHIFT) - scale_col : 0;
  auto fetch_scales = [&] {  // of the next stage
    if constexpr (W4) {
      if (scale_left >= S::kScaleLane) {
#pragma unroll
        for (int j = 0; j < S::kScaleLane; ++j) {
          asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(next_scale[j]) : "l"(scale_src + j));
          if constexpr (S::ZEROS)
            asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(next_zero[j]) : "l"(zero_src + j));
        }
      } else {
#pragma unroll
        for (int j = 0; j < S::kScaleLane; ++j) {
          next_scale[j] = 0;
          next_zero[j] = 8;
          if (j < scale_left) {
            asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(next_scale[j]) : "l"(scale_src + j));
            if constexpr (S::ZEROS)
              asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(next_zero[j]) : "l"(zero_src + j));
          }
        }
      }
      scale_src += S::kGroups;
      if constexpr (S::ZEROS) zero_src += S::kGroups;
      scale_left -= S::kGroups;
    }
  };
  auto keep_scales = [&](int i) {
    if constexpr (W4) {
      const int at = scale_row * S::kScalePitch + scale_col;
      uint16_t* set = reinterpret_cast<uint16_t*>(scale_sets + (i & 1) * S::kScaleBytes) + at;
      uint16_t* zset =
          reinterpret_cast<uint16_t*>(scale_sets + (2 + (i & 1)) * S::kScaleBytes) + at;
      if constexpr (S::kScaleLane == 1) {
        set[0] = (uint16_t)next_scale[0];
        if constexpr (S::ZEROS) zset[0] = (uint16_t)(Magic<T>::kBits + (next_zero[0] & 15));
      } else {
#pragma unroll
        for (int j = 0; j < S::kScaleLane; j += 2) {
          *reinterpret_cast<uint32_t*>(set + j) = next_scale[j] | next_scale[j + 1] << 16;
          if constexpr (S::ZEROS)
            *reinterpret_cast<uint32_t*>(zset + j) =
                Magic<T>::kBits * 0x10001u +
                ((next_zero[j] & 15) | (next_zero[j + 1] & 15) << 16);
        }
      }
    }
  };

  // Tokens of a panel: warp w brings rows w, w + 8, ..; 16-byte pieces lane, lane + 32. Held
  // in registers until the panel before is done with.
  constexpr int kPieces = S::kMaxPanel / 8 / 32;
  uint4 next_tokens[TILES][kPieces];
#pragma unroll
  for (int q = 0; q < TILES; ++q)
#pragma unroll
    for (int p = 0; p < kPieces; ++p) next_tokens[q][p] = make_uint4(0, 0, 0, 0);
  const uint16_t* token_row[TILES];
#pragma unroll
  for (int q = 0; q < TILES; ++q) {
    const int r = warp + 8 * q;
    int64_t at = -1;
    if (r < nrows) at = g.index ? g.index[begin + r] : begin + r;
    token_row[q] = at >= 0 && at < g.x_rows
                       ? static_cast<const uint16_t*>(g.x) + at * g.x_pitch
                       : nullptr;
  }
  auto fetch_tokens = [&](int k0) {
#pragma unroll
    for (int q = 0; q < TILES; ++q) {
      if (!token_row[q]) continue;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int k = k0 + (lane + 32 * p) * 8;
        next_tokens[q][p] = make_uint4(0, 0, 0, 0);
        if (k < k_end && (lane + 32 * p) * 8 < g.panel) {
          if (g.x_vec && k + 8 <= k_end) {
            next_tokens[q][p] = __ldg(reinterpret_cast<const uint4*>(token_row[q] + k));
          } else {
            uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (k + j < k_end) v[j / 2] |= (uint32_t)token_row[q][k + j] << (16 * (j & 1));
            next_tokens[q][p] = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
  };
  auto keep_tokens = [&](bool first) {
#pragma unroll
    for (int q = 0; q < TILES; ++q)
      if (token_row[q] || (first && q < tiles))  // rows of zeros stay
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          uint4 v = next_tokens[q][p];
          if (W4)  // pairs (0, 4), (1, 5), (2, 6), (3, 7)
            v = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                           __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
          if ((lane + 32 * p) * 8 < g.panel)
            *reinterpret_cast<uint4*>(tokens + (warp + 8 * q) * tpitch + (lane + 32 * p) * 16) = v;
        }
  };

  // acc is what the matrix instructions add to. They cut off at most 2^-23 of it each time, so
  // with weights of 16 bits a panel's sums (at most 32 times) go to `total`, in f32; 4-bit
  // weights' leave them at every scale group.
  float acc[TILES][4], total[TILES][4];
#pragma unroll
  for (int j = 0; j < TILES; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = total[j][i] = 0.0f;
  auto keep_sums = [&] {
    if constexpr (!W4) {
#pragma unroll
      for (int j = 0; j < TILES; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          total[j][i] += acc[j][i];
          acc[j][i] = 0.0f;
        }
    }
  };

#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) load_stage(i);
  fetch_scales();
  fetch_tokens(k_begin);
  keep_scales(0);

  uint32_t mask, magic;
  asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(mask));
  asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(Magic<T>::kBits * 0x10001u));
  int kp = g.panel;  // inner position in the panel
  int slot = 0;      // stage of the ring to multiply next
  for (int i = 0; i < stages; ++i, kp += S::kStageInner) {
    if (kp == g.panel) {
      kp = 0;
      if (i > 0) __syncthreads();
      keep_sums();
      keep_tokens(i == 0);
      __syncthreads();
      fetch_tokens(k_begin + i * S::kStageInner + g.panel);
    }
    load_stage(i + kRing - 1);
    if (i + 1 < stages) fetch_scales();
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
    __syncwarp();
    const uint8_t* st = ring + slot * kStageBytes;
    slot = slot + 1 == kRing ? 0 : slot + 1;
    if constexpr (W4) {
      const uint8_t* a_at = st + gq * kRowPitch + tq * 4;
      const uint8_t* b_at = tokens + gq * tpitch + (kp + tq * 8) * 2;
      const T* scales =
          reinterpret_cast<const T*>(scale_sets + (i & 1) * S::kScaleBytes);
      const uint16_t* zeros =
          reinterpret_cast<const uint16_t*>(scale_sets + (2 + (i & 1)) * S::kScaleBytes);
      constexpr int kSteps = (1 << SHIFT) / 32;  // of 32 in a scale group
#pragma unroll(TILES == 1 ? 4 : 1)
      for (int g2 = 0; g2 < S::kGroups; g2 += 2) {  // two scale groups: a word of each kind
        const int lo = gq * S::kScalePitch + g2, hi = lo + 8 * S::kScalePitch;
        const uint32_t sl2 = *reinterpret_cast<const uint32_t*>(scales + lo);
        const uint32_t sh2 = *reinterpret_cast<const uint32_t*>(scales + hi);
        uint32_t zl2 = 0, zh2 = 0;
        if constexpr (S::ZEROS) {
          zl2 = *reinterpret_cast<const uint32_t*>(zeros + lo);
          zh2 = *reinterpret_cast<const uint32_t*>(zeros + hi);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t zl = (Magic<T>::kBits + 8) * 0x10001u, zh = zl;
          if constexpr (S::ZEROS) {
            zl = __byte_perm(zl2, 0, h ? 0x3232 : 0x1010);
            zh = __byte_perm(zh2, 0, h ? 0x3232 : 0x1010);
          }
          float part[TILES][4];
#pragma unroll
          for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) part[n][q] = 0.0f;
#pragma unroll
          for (int i2 = 0; i2 < kSteps; ++i2) {
            const int j = (g2 + h) * kSteps + i2;
            const uint32_t wl = *reinterpret_cast<const uint32_t*>(a_at + j * 16);
            const uint32_t wh = *reinterpret_cast<const uint32_t*>(a_at + j * 16 + 8 * kRowPitch);
            uint32_t pl[4], ph[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              pl[q] = sub2<T>(and_or(wl >> (4 * q), mask, magic), zl);
              ph[q] = sub2<T>(and_or(wh >> (4 * q), mask, magic), zh);
            }
            const uint32_t a0[4] = {pl[0], ph[0], pl[1], ph[1]},
                           a1[4] = {pl[2], ph[2], pl[3], ph[3]};
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
              if (TILES == 1 || n < tiles) {
                const uint4 b = *reinterpret_cast<const uint4*>(b_at + n * 8 * tpitch + j * 64);
                mma_16816<T>(part[n], a0, b.x, b.y);
                mma_16816<T>(part[n], a1, b.z, b.w);
              }
            }
          }
          const float sl = half_of<T>(sl2, h), sh = half_of<T>(sh2, h);
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
      const uint32_t a_at = shared_addr(st) + (lane & 15) * kRowPitch + (lane >> 4) * 16;
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
    keep_scales(i + 1);
    __syncwarp();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  keep_sums();
  // partial sums as [row][output], over the tokens; with a split inner axis the blocks of
  // the cluster each add up and store a share of the rows
  __syncthreads();
  float* sums = reinterpret_cast<float*>(tokens);
#pragma unroll
  for (int n = 0; n < TILES; ++n)
    if (n < tiles) {
      float* at = sums + (n * 8 + 2 * tq) * kOutBlock + warp * 16 + gq;
      at[0] = W4 ? acc[n][0] : total[n][0];
      at[kOutBlock] = W4 ? acc[n][1] : total[n][1];
      at[8] = W4 ? acc[n][2] : total[n][2];
      at[kOutBlock + 8] = W4 ? acc[n][3] : total[n][3];
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

template <typename S>
cudaError_t launch_few_shape(FewArgs g, cudaStream_t st) {
  static std::atomic<bool> ready[kMaxDevices];  // the kernel's shared memory limit is raised
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    err = cudaFuncSetAttribute(k_grouped_few<S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               S::total(S::kMaxPanel));
    if (err != cudaSuccess) return err;
    ready[dev].store(true, std::memory_order_release);
  }
  const int64_t blocks = (g.outer + kOutBlock - 1) / kOutBlock;
  // every group of rows, the two without an expert among them, has one ragged item at most
  const int64_t items = std::min<int64_t>(g.experts + 2, g.rows) + g.rows / S::kRows;
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
  cfg.dynamicSmemBytes = (size_t)S::total(g.panel);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_grouped_few<S>, g);
}

template <typename T, int SHIFT, bool ZEROS, int ALIGN>
cudaError_t launch_few_rows(const FewArgs& g, cudaStream_t st) {
  // Items of 8 rows while few experts can have more: no test for absent column tiles in the
  // inner loop, and the tokens of twice the inner length in shared memory.
  return g.rows <= 4 * (int64_t)g.experts || g.rows <= 8
             ? launch_few_shape<FewShape<T, 1, SHIFT, ZEROS, ALIGN>>(g, st)
             : launch_few_shape<FewShape<T, 4, SHIFT, ZEROS, ALIGN>>(g, st);
}

template <typename T>
cudaError_t launch_few_typed(const FewArgs& g, int group_size, int align, cudaStream_t st) {
  if (group_size == 0) {
    if (align == 16) return launch_few_rows<T, 0, false, 16>(g, st);
    if (align == 4) return launch_few_rows<T, 0, false, 4>(g, st);
    return launch_few_rows<T, 0, false, 2>(g, st);
  }
  if (group_size == 32)
    return g.zeros ? launch_few_rows<T, 5, true, 16>(g, st)
                   : launch_few_rows<T, 5, false, 16>(g, st);
  if (group_size == 64)
    return g.zeros ? launch_few_rows<T, 6, true, 16>(g, st)
                   : launch_few_rows<T, 6, false, 16>(g, st);
  return g.zeros ? launch_few_rows<T, 7, true, 16>(g, st)
                 : launch_few_rows<T, 7, false, 16>(g, st);
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
  int align = 16;
  if (c.group_size == 0) {
    g.w_pitch = (int64_t)c.inner * 2;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(c.w) | (uintptr_t)g.w_pitch;
    align = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
  } else {
    g.w_pitch = (c.inner + 31) / 32 * 16;
    g.scales = c.scales;
    g.zeros = c.zeros;
    g.groups = (c.inner + c.group_size - 1) / c.group_size;
  }
  return c.dtype == LGBM_B200_DTYPE_F16
             ? launch_few_typed<__half>(g, c.group_size, align, st)
             : launch_few_typed<__nv_bfloat16>(g, c.group_size, align, st);
}

}  // namespace experts
}  // namespace lgbm_b200
