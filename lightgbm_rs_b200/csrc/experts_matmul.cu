// Matrix products grouped by expert, forward and both gradients, on the 5th-generation
// tensor cores.
//
//   FORWARD   y[r, n]     = sum_k x[r, k] w[e(r), n, k]
//   INPUT     dx[r, k]    = sum_n dy[r, n] w[e(r), n, k]
//   WEIGHT    dw[e, n, k] = sum_{r in group e} dy[r, n] x[r, k]
//
// Rows are grouped: group e is rows offsets[e] .. offsets[e + 1]. All three are one kernel:
// D (128 x BN, f32 in tensor memory) += A (128 x 64) B (64 x BN) over blocks of 64 of the
// reduction; only the operands' layouts differ. An operand whose reduction axis is contiguous
// in memory is staged K-major, else MN-major (panels of 64 columns), both with 128-byte
// swizzle, so nothing is transposed on the way. A persistent grid walks the tiles of all
// groups; one warp issues TMA loads, one issues the matrix instructions, four write results
// out of one half of tensor memory while the next tile accumulates in the other.
//
// Ragged ends. FORWARD / INPUT: a tile's rows past its group's end are computed from the next
// group's rows and not stored (a row of A only reaches its own row of D). Rows past the last
// group form one more group without a reduction: zeros. WEIGHT: the reduction itself ends
// inside a block; the rows past the end are zeroed in both operands in shared memory (in
// both, so that an infinity or NaN of the next group cannot make 0 * inf).
#include <algorithm>
#include <mutex>

#include <cuda.h>  // types of the tensor map; the encoder is looked up at run time

#include "experts.cuh"

namespace lgbm_b200 {
namespace experts {
namespace {

constexpr int kMatThreads = 192;   // warp 0 loads, warp 1 multiplies, warps 2..5 store
constexpr int kTileM = 128;
constexpr int kTileK = 64;         // 128 bytes of a 16-bit type: one swizzle row
constexpr int kStoreBytes = 4 * 32 * 128;  // one 32 x 128 B staging block a storing warp
constexpr int kBand = 16;          // row tiles of a band, see tile_of
constexpr uint64_t kWaitNs = 2000000000;

enum Mode { FORWARD = 0, INPUT = 1, WEIGHT = 2 };

struct MatArgs {
  const int32_t* offsets;
  int32_t experts;
  int32_t cols;        // columns of D in a group
  int32_t drows;       // WEIGHT: rows of D in a group
  int32_t reduction;   // FORWARD, INPUT: length of the reduction
  int32_t out_kind;    // LGBM_B200_DTYPE_*
  int32_t vec;         // 16-byte stores
  uint32_t idesc;
  int64_t rows;
  int64_t out_pitch;
  void* out;
  uint32_t* error;
};

// Set by a kernel whose bounded wait ran out; lgbm_b200_experts_errors reads and clears it.
__device__ uint32_t g_matmul_error;

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// A whole warp waits; bounded: false, in every lane, when two seconds were not enough for one.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  bool done = bar_try(bar, parity);
  if (!done) {
    const uint64_t start = now_ns();
    do {
#pragma unroll 1
      for (int i = 0; i < 32 && !done; ++i) done = bar_try(bar, parity);
    } while (!done && now_ns() - start < kWaitNs);
  }
  return __all_sync(0xFFFFFFFFu, done);
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
// 32 lanes x 32 columns of f32 of this warp's quarter of tensor memory.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
        "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle (layout 2), version 1. `lead` and
// `stride` in bytes: K-major, `stride` between groups of 8 rows; MN-major, `lead` between
// panels of 64 columns and `stride` between groups of 8 reduction rows.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lead >> 4) << 16) |
         ((uint64_t)(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

struct Tile {
  int32_t group;
  int32_t m0;      // first row of D: of all rows (FORWARD, INPUT), of the group (WEIGHT)
  int32_t m_end;   // rows of D end here
  int32_t n0;
  int32_t red0;    // WEIGHT: first row of the reduction
  int32_t red;     // length of the reduction
};

// Tile `t` of a group of mt x nt tiles: bands of kBand row tiles, column by column inside a
// band, so that the CTAs at work at one time share a few row tiles and a few column tiles.
__device__ __forceinline__ void tile_of(int t, int mt, int nt, int& m, int& n) {
  const int band = t / (kBand * nt), r = t - band * kBand * nt;
  const int h = min(kBand, mt - band * kBand);
  n = r / h;
  m = band * kBand + (r - n * h);
}

template <int MODE, int BN>
struct Shape {
  static constexpr int kStageBytes = (kTileM + BN) * 128;
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int kTmemCols = 2 * BN;  // two accumulators
  static constexpr int kSmem =
      1024 + kStages * kStageBytes + kStoreBytes + 4 * (kMaxExperts + 2) + 256;
};

template <int MODE, int BN>
__global__ void __launch_bounds__(kMatThreads, 1)
    k_grouped_matmul(const __grid_constant__ CUtensorMap map_a,
                     const __grid_constant__ CUtensorMap map_b, const MatArgs g) {
  using S = Shape<MODE, BN>;
  constexpr int kStages = S::kStages;
  constexpr uint32_t kABytes = kTileM * 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t base = smem_addr(smem);
  const uint32_t store_base = base + kStages * S::kStageBytes;
  int32_t* cum = reinterpret_cast<int32_t*>(smem + kStages * S::kStageBytes + kStoreBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(
      (reinterpret_cast<uintptr_t>(cum + kMaxExperts + 2) + 15) & ~(uintptr_t)15);
  const uint32_t full = smem_addr(bars), empty = full + 8 * kStages,
                 acc_full = empty + 8 * kStages, acc_empty = acc_full + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        bar_init(full + 8 * i, 1);
        bar_init(empty + 8 * i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        bar_init(acc_full + 8 * i, 1);
        bar_init(acc_empty + 8 * i, 4);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    }
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "r"((uint32_t)S::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == 2) {
    // first tile of every group; FORWARD and INPUT have one group more, the rows past the
    // last offset
    const int groups = MODE == WEIGHT ? g.experts : g.experts + 1;
    const int nt = (g.cols + BN - 1) / BN;
    int32_t carry = 0;
    for (int i0 = 0; i0 < groups; i0 += 32) {
      const int i = i0 + lane;
      int32_t v = 0;
      if (i < groups) {
        if (MODE == WEIGHT) {
          v = (g.drows + kTileM - 1) / kTileM * nt;
        } else {
          int64_t b = min(max((int64_t)g.offsets[i], (int64_t)0), g.rows);
          int64_t e = i < g.experts ? min(max((int64_t)g.offsets[i + 1], b), g.rows) : g.rows;
          v = (int32_t)((e - b + kTileM - 1) / kTileM) * nt;
        }
      }
      int32_t s = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int32_t o = __shfl_up_sync(0xFFFFFFFFu, s, d);
        if (lane >= d) s += o;
      }
      if (i < groups) cum[i] = carry + s - v;
      carry += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
    if (lane == 0) cum[groups] = carry;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int groups = MODE == WEIGHT ? g.experts : g.experts + 1;
  const int tiles = cum[groups];
  const int nt = (g.cols + BN - 1) / BN;

  auto decode = [&](int t) {
    int lo = 0, hi = groups;  // the last group that starts at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] <= t) lo = mid; else hi = mid;
    }
    int64_t b = min(max((int64_t)g.offsets[lo], (int64_t)0), g.rows);
    int64_t e = lo < g.experts ? min(max((int64_t)g.offsets[lo + 1], b), g.rows) : g.rows;
    Tile r;
    r.group = lo;
    int m, n;
    const int drows = MODE == WEIGHT ? g.drows : (int)(e - b);
    tile_of(t - cum[lo], (drows + kTileM - 1) / kTileM, nt, m, n);
    r.n0 = n * BN;
    if (MODE == WEIGHT) {
      r.m0 = m * kTileM;
      r.m_end = g.drows;
      r.red0 = (int)b;
      r.red = (int)(e - b);
    } else {
      r.m0 = (int)b + m * kTileM;
      r.m_end = (int)e;
      r.red0 = 0;
      r.red = lo < g.experts ? g.reduction : 0;
    }
    return r;
  };

  bool ok = true;
  if (warp == 0) {
    uint32_t it = 0;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      const Tile r = decode(t);
      for (int k0 = 0; k0 < r.red; k0 += kTileK, ++it) {
        const uint32_t s = it % kStages;
        if (it >= kStages && !(ok = bar_wait(empty + 8 * s, (it / kStages - 1) & 1))) break;
        if (elect_one()) {
          const uint32_t a = base + s * S::kStageBytes, b = a + kABytes, bar = full + 8 * s;
          bar_expect(bar, S::kStageBytes);
          if (MODE == WEIGHT) {
#pragma unroll
            for (int j = 0; j < kTileM / 64; ++j)
              tma_load_2d(a + j * 8192, &map_a, r.m0 + 64 * j, r.red0 + k0, bar);
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              tma_load_2d(b + j * 8192, &map_b, r.n0 + 64 * j, r.red0 + k0, bar);
          } else {
            tma_load_2d(a, &map_a, k0, r.m0, bar);
            if (MODE == FORWARD) {
              tma_load_3d(b, &map_b, k0, r.n0, r.group, bar);
            } else {
#pragma unroll
              for (int j = 0; j < BN / 64; ++j)
                tma_load_3d(b + j * 8192, &map_b, r.n0 + 64 * j, k0, r.group, bar);
            }
          }
        }
        __syncwarp();
      }
    }
    // no copy may be in flight when the CTA ends: a load whose block nobody multiplied
    // (another warp gave up) has still landed before the CTA leaves
    if (!ok)
      for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
        bar_wait(full + 8 * (i % kStages), (i / kStages) & 1);
  } else if (warp == 1) {
    uint32_t it = 0, tile = 0;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      const Tile r = decode(t);
      if (r.red == 0) continue;
      const uint32_t acc = tile & 1, d = tmem + acc * BN;
      if (tile >= 2 && !(ok = bar_wait(acc_empty + 8 * acc, (tile / 2 - 1) & 1))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (int k0 = 0; k0 < r.red; k0 += kTileK, ++it) {
        const uint32_t s = it % kStages;
        if (!(ok = bar_wait(full + 8 * s, (it / kStages) & 1))) break;
        const uint32_t a = base + s * S::kStageBytes, b = a + kABytes;
        int steps = kTileK / 16;
        if (MODE == WEIGHT && r.red - k0 < kTileK) {
          // the group ends inside this block: whole steps past it are left out, and the rows
          // between its end and the last step's are zeroed in every panel
          const int valid = r.red - k0;
          steps = (valid + 15) / 16;
          const int rest = steps * 16 - valid;
          constexpr int kPanels = (kTileM + BN) / 64;
          for (int i = lane; i < rest * kPanels * 8; i += 32) {
            const int panel = i / (rest * 8), row = i / 8 % rest;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             a + panel * 8192 + (valid + row) * 128 + (i & 7) * 16),
                         "r"(0)
                         : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        if (elect_one()) {
          for (int k = 0; k < steps; ++k) {
            // 16 of the reduction: 32 bytes along a K-major row, 16 rows of an MN-major panel
            const uint64_t da = MODE == WEIGHT ? smem_desc(a + k * 2048, 8192, 1024)
                                               : smem_desc(a + k * 32, 16, 1024);
            const uint64_t db = MODE == FORWARD ? smem_desc(b + k * 32, 16, 1024)
                                                : smem_desc(b + k * 2048, 8192, 1024);
            mma_f16(d, da, db, g.idesc, k0 > 0 || k > 0);
          }
          mma_commit(empty + 8 * s);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) mma_commit(acc_full + 8 * acc);
      __syncwarp();
      ++tile;
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t stage = store_base + (warp - 2) * 4096;
    const int bytes = g.out_kind == LGBM_B200_DTYPE_F32 ? 4 : 2;
    const int per_chunk = 128 / bytes;  // columns of a 128-byte staging row
    uint32_t tile = 0;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      const Tile r = decode(t);
      const uint32_t acc = tile & 1;
      if (r.red > 0) {
        if (!(ok = bar_wait(acc_full + 8 * acc, (tile / 2) & 1))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      const int row0 = r.m0 + quarter * 32;
      char* out = static_cast<char*>(g.out);
      if (MODE == WEIGHT) out += (int64_t)r.group * g.drows * g.out_pitch * bytes;
      const int ncols = min(BN, g.cols - r.n0);
      for (int c0 = 0; c0 < ncols; c0 += per_chunk) {
        // this lane's row into the staging block, 16-byte pieces swizzled by row
        for (int h = 0; h < per_chunk; h += 32) {
          uint32_t v[32];
          if (r.red > 0) {
            tmem_load32(tmem + acc * BN + ((uint32_t)(quarter * 32) << 16) + c0 + h, v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0;
          }
          if (g.out_kind == LGBM_B200_DTYPE_F32) {
#pragma unroll
            for (int p = 0; p < 8; ++p)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                               stage + lane * 128 + ((p ^ (lane & 7)) << 4)),
                           "r"(v[4 * p]), "r"(v[4 * p + 1]), "r"(v[4 * p + 2]), "r"(v[4 * p + 3])
                           : "memory");
          } else {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x = __uint_as_float(v[2 * i]), y = __uint_as_float(v[2 * i + 1]);
              if (g.out_kind == LGBM_B200_DTYPE_BF16) {
                const __nv_bfloat162 q = __floats2bfloat162_rn(x, y);
                w[i] = *reinterpret_cast<const uint32_t*>(&q);
              } else {
                const __half2 q = __floats2half2_rn(x, y);
                w[i] = *reinterpret_cast<const uint32_t*>(&q);
              }
            }
#pragma unroll
            for (int p = 0; p < 4; ++p)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                               stage + lane * 128 + (((h / 8 + p) ^ (lane & 7)) << 4)),
                           "r"(w[4 * p]), "r"(w[4 * p + 1]), "r"(w[4 * p + 2]), "r"(w[4 * p + 3])
                           : "memory");
          }
        }
        __syncwarp();
        const int n = min(per_chunk, ncols - c0);
        char* dst = out + ((int64_t)row0 * g.out_pitch + r.n0 + c0) * bytes;
        const int nrows = min(32, r.m_end - row0);
        if (g.vec && n * bytes % 16 == 0) {
          // 8 lanes a row, 4 rows a store
          for (int i = lane >> 3; i < nrows; i += 4) {
            const int p = lane & 7;
            if (p * 16 < n * bytes) {
              uint32_t w[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                           : "r"(stage + i * 128 + ((p ^ (i & 7)) << 4))
                           : "memory");
              *reinterpret_cast<uint4*>(dst + (int64_t)i * g.out_pitch * bytes + p * 16) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        } else {
          for (int i = 0; i < nrows; ++i)
            for (int c = lane; c < n; c += 32) {
              const uint32_t at = stage + i * 128 + (((c * bytes >> 4) ^ (i & 7)) << 4) +
                                  (c * bytes & 15);
              if (bytes == 4) {
                uint32_t w;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
                *reinterpret_cast<uint32_t*>(dst + ((int64_t)i * g.out_pitch + c) * 4) = w;
              } else {
                uint16_t w;
                asm volatile("ld.shared.b16 %0, [%1];" : "=h"(w) : "r"(at) : "memory");
                *reinterpret_cast<uint16_t*>(dst + ((int64_t)i * g.out_pitch + c) * 2) = w;
              }
            }
        }
        __syncwarp();
      }
      if (r.red > 0) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(acc_empty + 8 * acc);
        ++tile;
      }
    }
  }
  if (!ok && lane == 0) atomicOr(g.error, 1u);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"((uint32_t)S::kTmemCols));
}

// Rows copied to a pitch that TMA can walk: dst[r] = src[index ? index[r] : r], the columns
// between `width` and `dst_pitch` zero; a row whose index is outside is zero.
__global__ void __launch_bounds__(256)
    k_stage_rows(const uint16_t* src, int64_t src_rows, int64_t rows, int width, int64_t pitch,
                 const int32_t* index, uint16_t* dst, int64_t dst_pitch, int words) {
  const int per_row = (int)(dst_pitch / 8);
  const int64_t total = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row;
    const int c = (int)(i - r * per_row) * 8;
    const int64_t at = index ? index[r] : r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (at >= 0 && at < src_rows) {
      const uint16_t* p = src + at * pitch + c;
      if (words == 8 && c + 8 <= width) {
        v = *reinterpret_cast<const uint4*>(p);
      } else if (words >= 4 && c + 8 <= width) {
        const uint2 lo = *reinterpret_cast<const uint2*>(p);
        const uint2 hi = *reinterpret_cast<const uint2*>(p + 4);
        v = make_uint4(lo.x, lo.y, hi.x, hi.y);
      } else {
        uint16_t e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = c + j < width ? p[j] : (uint16_t)0;
        v = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16,
                       e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
      }
    }
    *reinterpret_cast<uint4*>(dst + r * dst_pitch + c) = v;
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// A tensor of 16-bit elements, innermost axis first; boxes of 64 x `box1` elements, 128-byte
// swizzle, zeros outside the tensor.
bool encode(CUtensorMap* map, int32_t dtype, const void* base, int rank, const int64_t* dims,
            const int64_t* pitches, int box1) {
  cuuint64_t d[3], s[2];
  cuuint32_t box[3] = {64, (cuuint32_t)box1, 1}, step[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) d[i] = (cuuint64_t)dims[i];
  for (int i = 0; i + 1 < rank; ++i) s[i] = (cuuint64_t)pitches[i] * 2;
  const EncodeTiled fn = encoder();
  return fn && fn(map,
                  dtype == LGBM_B200_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  (cuuint32_t)rank, const_cast<void*>(base), d, s, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a launch needs to know of the current device, looked up once a device.
constexpr int kMaxDevices = 64;
struct DeviceInfo {
  std::mutex mu;
  int sms = 0;
  uint32_t* error = nullptr;
  uint32_t smem_set = 0;  // instantiations whose shared memory limit is raised, one bit each
};
DeviceInfo g_devices[kMaxDevices];

template <int MODE, int BN>
cudaError_t launch_tiles(const CUtensorMap& a, const CUtensorMap& b, MatArgs g,
                         int64_t most_tiles, cudaStream_t st) {
  using S = Shape<MODE, BN>;
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  {
    DeviceInfo& d = g_devices[dev];
    std::lock_guard<std::mutex> lock(d.mu);
    if (!d.error) {
      void* p = nullptr;
      err = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
      if (err == cudaSuccess) err = cudaGetSymbolAddress(&p, g_matmul_error);
      if (err != cudaSuccess) return err;
      d.error = static_cast<uint32_t*>(p);
    }
    constexpr uint32_t bit = 1u << (MODE * 3 + (BN == 64 ? 0 : BN == 128 ? 1 : 2));
    if (!(d.smem_set & bit)) {
      err = cudaFuncSetAttribute(k_grouped_matmul<MODE, BN>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
      if (err != cudaSuccess) return err;
      d.smem_set |= bit;
    }
    g.error = d.error;
    sms = d.sms;
  }
  const int grid = (int)std::min<int64_t>(sms, most_tiles);
  k_grouped_matmul<MODE, BN><<<grid, kMatThreads, S::kSmem, st>>>(a, b, g);
  return cudaGetLastError();
}

// An operand as TMA can read it: 16-byte base and pitches, or a copy in the workspace.
struct Operand {
  const void* p;
  int64_t pitch;
};

bool walkable(const void* p, int64_t pitch) { return aligned16(p) && pitch % 8 == 0; }
int64_t padded(int64_t width) { return (width + 7) / 8 * 8; }
int64_t copy_bytes(int64_t rows, int64_t width) {
  return (rows * padded(width) * 2 + 255) / 256 * 256;
}

cudaError_t stage(Operand& o, int64_t src_rows, int64_t rows, int width, const int32_t* index,
                  char*& workspace, cudaStream_t st) {
  const int64_t dst_pitch = padded(width);
  uint16_t* dst = reinterpret_cast<uint16_t*>(workspace);
  workspace += copy_bytes(rows, width);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(o.p) | (uintptr_t)(o.pitch * 2);
  const int words = bits % 16 == 0 ? 8 : bits % 8 == 0 ? 4 : 1;
  const int64_t want = (rows * (dst_pitch / 8) + 255) / 256;
  k_stage_rows<<<(unsigned)std::min<int64_t>(want, 1 << 20), 256, 0, st>>>(
      static_cast<const uint16_t*>(o.p), src_rows, rows, width, o.pitch, index, dst, dst_pitch,
      words);
  o.p = dst;
  o.pitch = dst_pitch;
  return cudaGetLastError();
}

uint32_t instruction(int32_t dtype, bool a_mn, bool b_mn, int bn) {
  const uint32_t type = dtype == LGBM_B200_DTYPE_BF16 ? 1 : 0;
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn << 15) |
         ((uint32_t)b_mn << 16) | ((uint32_t)(bn / 8) << 17) | ((uint32_t)(kTileM / 16) << 24);
}

template <int MODE>
cudaError_t run_tiles(const Operand& a, int64_t a_width, int64_t rows, const Operand& b,
                      int64_t b_width, int32_t dtype, MatArgs g, cudaStream_t st) {
  const int bytes = elem_size(g.out_kind);
  g.vec = aligned16(g.out) && g.out_pitch * bytes % 16 == 0 &&
          (int64_t)g.drows * g.out_pitch * bytes % 16 == 0;
  auto go = [&](auto bn_c) -> cudaError_t {
    constexpr int BN = decltype(bn_c)::value;
    CUtensorMap ma, mb;
    const int64_t da[3] = {a_width, rows, 1}, pa[2] = {a.pitch, 0};
    bool fine = encode(&ma, dtype, a.p, 2, da, pa, MODE == WEIGHT ? 64 : kTileM);
    if (MODE == WEIGHT) {
      const int64_t db[3] = {b_width, rows, 1}, pb[2] = {b.pitch, 0};
      fine = fine && encode(&mb, dtype, b.p, 2, db, pb, 64);
    } else {
      const int64_t n = MODE == FORWARD ? g.cols : g.reduction;
      const int64_t db[3] = {b_width, n, g.experts}, pb[2] = {b.pitch, b.pitch * n};
      fine = fine && encode(&mb, dtype, b.p, 3, db, pb, MODE == FORWARD ? BN : 64);
    }
    if (!fine) return cudaErrorInvalidValue;
    g.idesc = instruction(dtype, MODE == WEIGHT, MODE != FORWARD, BN);
    const int64_t nt = (g.cols + BN - 1) / BN;
    const int64_t most = MODE == WEIGHT
                             ? (int64_t)g.experts * ((g.drows + kTileM - 1) / kTileM) * nt
                             : (rows / kTileM + g.experts + 1) * nt;
    return launch_tiles<MODE, BN>(ma, mb, g, most, st);
  };
  if (g.cols <= 64) return go(std::integral_constant<int, 64>());
  if (g.cols <= 128) return go(std::integral_constant<int, 128>());
  return go(std::integral_constant<int, 256>());
}

}  // namespace

// Few rows an expert: the forward product streams the weights instead (experts_few.cu).
bool few_rows(const MatmulCall& c) { return c.mode == 0 && c.rows <= 16 * (int64_t)c.experts; }

int64_t matmul_workspace(const MatmulCall& c) {
  int64_t n = 0;
  if (few_rows(c)) return 0;
  if (c.mode != 1 && (c.index || !walkable(c.x, c.x_pitch))) n += copy_bytes(c.rows, c.inner);
  if (c.mode != 0 && !walkable(c.dy, c.dy_pitch)) n += copy_bytes(c.rows, c.outer);
  if (c.mode != 2 && !(aligned16(c.w) && c.inner % 8 == 0))
    n += copy_bytes((int64_t)c.experts * c.outer, c.inner);
  return n;
}

cudaError_t launch_matmul(const MatmulCall& c, void* workspace, cudaStream_t st) {
  if (few_rows(c)) {
    FewCall f{};
    f.dtype = c.dtype;
    f.x = c.x;
    f.x_rows = c.x_rows;
    f.x_pitch = c.x_pitch;
    f.index = c.index;
    f.w = c.w;
    f.offsets = c.offsets;
    f.rows = c.rows;
    f.experts = c.experts;
    f.inner = c.inner;
    f.outer = c.outer;
    f.y = c.out;
    return launch_few(f, st);
  }
  char* ws = static_cast<char*>(workspace);
  MatArgs g{};
  g.offsets = c.offsets;
  g.experts = c.experts;
  g.rows = c.rows;
  g.out = c.out;
  g.out_kind = c.out_dtype;
  Operand x{c.x, c.x_pitch}, dy{c.dy, c.dy_pitch}, w{c.w, c.inner};
  cudaError_t err = cudaSuccess;
  if (c.mode != 1 && (c.index || !walkable(c.x, c.x_pitch)))
    err = stage(x, c.x_rows, c.rows, c.inner, c.index, ws, st);
  if (err == cudaSuccess && c.mode != 0 && !walkable(c.dy, c.dy_pitch))
    err = stage(dy, c.rows, c.rows, c.outer, nullptr, ws, st);
  if (err == cudaSuccess && c.mode != 2 && !(aligned16(c.w) && c.inner % 8 == 0))
    err = stage(w, (int64_t)c.experts * c.outer, (int64_t)c.experts * c.outer, c.inner, nullptr,
                ws, st);
  if (err != cudaSuccess) return err;
  if (c.mode == 0) {
    g.cols = c.outer;
    g.reduction = c.inner;
    g.out_pitch = c.outer;
    return run_tiles<FORWARD>(x, c.inner, c.rows, w, c.inner, c.dtype, g, st);
  }
  if (c.mode == 1) {
    g.cols = c.inner;
    g.reduction = c.outer;
    g.out_pitch = c.inner;
    return run_tiles<INPUT>(dy, c.outer, c.rows, w, c.inner, c.dtype, g, st);
  }
  g.cols = c.inner;
  g.drows = c.outer;
  g.out_pitch = c.inner;
  return run_tiles<WEIGHT>(dy, c.outer, c.rows, x, c.inner, c.dtype, g, st);
}

cudaError_t read_matmul_errors(uint32_t* bits) {
  cudaError_t err = cudaMemcpyFromSymbol(bits, g_matmul_error, sizeof(*bits));
  const uint32_t zero = 0;
  if (err == cudaSuccess && *bits)
    err = cudaMemcpyToSymbol(g_matmul_error, &zero, sizeof(zero));
  return err;
}

}  // namespace experts
}  // namespace lgbm_b200
