// Matrix products grouped by expert, forward and both gradients, on the 5th-generation
// tensor cores.
//
//   FORWARD   y[r, n]     = sum_k x[r, k] w[e(r), n, k]
//   INPUT     dx[r, k]    = sum_n dy[r, n] w[e(r), n, k]
//   WEIGHT    dw[e, n, k] = sum_{r in group e} dy[r, n] x[r, k]
//
// Rows are grouped: group e is rows offsets[e] .. offsets[e + 1]. All three are one kernel:
// D (f32 in tensor memory) += A B over blocks of 64 of the reduction; only the operands'
// layouts differ. An operand whose reduction axis is contiguous in memory is staged K-major,
// else MN-major (panels of 64 columns), both with 128-byte swizzle, so nothing is transposed
// on the way. A persistent grid walks the tiles of all groups; in every CTA one warp issues
// TMA loads, one the matrix instructions, and eight write results out of one half of tensor
// memory while the next tile accumulates in the other.
//
// Pairs. A 128 x 256 tile of one CTA takes in 48 KB for each 512 cycles of matrix work: the
// SMs together ask more of L2 than it gives. Two CTAs of a cluster therefore share a
// 256 x 256 tile (cta_group::2): each loads half of A and half of B, 32 KB, and the even one
// multiplies for both. Single CTAs remain for groups of few rows and for few columns.
//
// Operands that TMA cannot walk (x read through an index; rows that do not start at 16 bytes:
// 700 features are 1400 bytes) are first copied to rows that it can (k_stage_rows), which
// costs their bytes twice more. Two ways without that copy were built and measured on 65536
// gathered rows of 2048 against 4096 outputs, where the product takes 0.77 ms and the copy
// 0.08: TMA gathers of four rows took about 20 cycles a row of 128 bytes (2.5 ms in all), and
// six warps of asynchronous 16-byte copies, each waiting out its own block's latency, 1.5.
//
// Ragged ends. FORWARD / INPUT: a tile's rows past its group's end are computed from the next
// group's rows and not stored (a row of A only reaches its own row of D). Rows past the last
// group and rows before the first form two more groups without a reduction: zeros. WEIGHT: the
// reduction itself ends inside a block. Steps of 16 past the end are left out, and in the last
// step the rows past it are overwritten with zeros in shared memory, in both operands: an
// infinity or NaN of the next group cannot make 0 * inf. In a pair each CTA's second warp does
// that to its own half and the odd one tells the even one. (Gathering that block's rows one by
// one, with zeros from TMA for those outside, took five times a block's time, once a tile.)
//
// Precision. The tensor cores cut a sum off when they add to it: 16 terms at a time, at most
// 2^-23 of the sum each time. With terms of one sign nearly all of that was measured at every
// addition: 1.6e-3 of the result at 2^18 terms in one piece, three times f16's unit roundoff.
// A reduction is therefore accumulated in runs, which the storing warps add up in f32 (a
// rounding of 2^-24 a run). Results of 16 bits: runs of 4096, which cut off at most 3.1e-5, a
// sixteenth of f16's unit roundoff. The second run on goes to the other half of tensor memory
// and is added to the first half there, while the tensor cores wait (16 groups of 4096 rows on
// average, 4096 x 2048: 2 %). Holding the sums in registers instead cost the tiles of one run
// up to 45 % (255 experts of 129 x 700: the code of their odd stores spilled). A weight
// gradient kept in f32 would show runs of that length, so there they are of 768, alternate
// between the halves without a wait, and the sums stay in the registers of twice as many
// storing warps: 7e-7 of the result up to 2^16 rows of random sign (1.3e-6 of one sign),
// 1.0e-6 (1.4e-6) at 2^20, against 1.7e-5 (1.2e-4) of cuBLAS's f32 product.
//
// Measured, loops on a warm GPU, equal groups: 65536 rows, 16 experts of 4096 x 2048: y 0.76
// to 0.91 ms as the power cap lets the clock (1.2 to 1.4 PFLOP/s), dx 0.86 to 0.91, dw 0.90 to
// 0.92 (bf16) and 1.04 to 1.06 (f32); cuBLAS's batched product of the same size 0.81 to 0.85,
// 0.81, 0.80 to 0.84. 8192 rows, 8 experts of 4096 x 1024: 58, 63 to 71, 67 us (f32 90)
// against 57 to 67, 51 to 55, 60 to 70; tensor pipe 52 to 63 % busy; the rest is the last
// wave, tiles that groups of 1024 and a few rows leave partly empty, and loads at the 64 bytes
// a cycle that an SM takes from L2. 40009 rows, 255 experts of 136 x 704: y 32, dx 49, dw 48
// and 59 us, 2 to 3 TB/s: two or three blocks of reduction a tile, bound by writing tiles out.
// (Dealing dw's tiles out longest group first gained nothing.)
#include <algorithm>
#include <atomic>
#include <mutex>

#include <cuda.h>  // types of the tensor map; the encoder is looked up at run time

#include "experts.cuh"
#include "experts_parts.h"
#include "wait_budget.h"

namespace lgbm_b200 {
namespace experts {
namespace {

constexpr int kTileM = 128;       // rows of D of a CTA
constexpr int kTileK = 64;         // 128 bytes of a 16-bit type: one swizzle row
constexpr int kStoreRow = 64;      // bytes of a row in a storing warp's staging block
constexpr int kBandRows = 2048;    // rows of D of a band, see tile_of
// Entries of the table of groups: the rows before the first expert's, the experts, the rows past
// the last one's, the end.
constexpr int kGroupSlots = kMaxExperts + 3;

enum Mode { FORWARD = 0, INPUT = 1, WEIGHT = 2, WEIGHT_F32 = 3 };

struct MatArgs {
  const int32_t* offsets;
  int32_t experts;     // groups: WEIGHT has `parts` of each expert's
  int32_t parts;
  int32_t cols;        // columns of D in a group
  int32_t drows;       // WEIGHT: rows of D in a group
  int32_t reduction;   // FORWARD, INPUT: length of the reduction
  int32_t out_kind;    // LGBM_B200_DTYPE_*
  int32_t unit;        // bytes of a store: what the alignment of every row of D allows
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
// Arrives at the barrier at this address of the cluster's first CTA.
__device__ __forceinline__ uint32_t leader_addr(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
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
// A whole warp waits; bounded: false, in every lane, when two seconds on the device were not
// enough for one.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  bool done = bar_try(bar, parity);
  if (!done) {
    WaitBudget budget(now_ns());
    do {
#pragma unroll 1
      for (int i = 0; i < 32 && !done; ++i) done = bar_try(bar, parity);
    } while (!done && budget.spend(now_ns()));
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
// TMA loads into this CTA's shared memory. In a pair the barrier is the first CTA's.
template <int CTAS>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        bool accumulate) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// Arrives, when the matrix work issued so far is done, at this barrier of every CTA at it.
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
}
// 32 lanes x 16 columns of f32 of this warp's quarter of tensor memory, and 32 columns.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
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
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 "
      "[%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Two f32 as one word of 16-bit values.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(uint32_t lo, uint32_t hi) {
  const float x = __uint_as_float(lo), y = __uint_as_float(hi);
  if constexpr (BF16) {
    const __nv_bfloat162 q = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&q);
  } else {
    const __half2 q = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&q);
  }
}
__device__ __forceinline__ void store_piece(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                            uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle (layout 2), version 1. `lead` and
// `stride` in bytes: K-major, `stride` between groups of 8 rows; MN-major, `lead` between
// panels of 64 columns and `stride` between groups of 8 reduction rows.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lead >> 4) << 16) |
         ((uint64_t)(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

struct Tile {
  int32_t expert;
  int32_t m0;      // first row of D: of all rows (FORWARD, INPUT), of the group (WEIGHT)
  int32_t m_end;   // rows of D end here
  int32_t n0;
  int32_t red0;    // WEIGHT: first row of the reduction
  int32_t red;     // length of the reduction
};

// Tile `t` of a group of mt x nt tiles: bands of `band` row tiles, column by column inside a
// band, so that the CTAs at work at one time share a few row tiles and a few column tiles.
__device__ __forceinline__ void tile_of(int t, int mt, int nt, int band, int& m, int& n) {
  const int b = t / (band * nt), r = t - b * band * nt;
  const int h = min(band, mt - b * band);
  n = r / h;
  m = b * band + (r - n * h);
}

// CTAS CTAs share a tile of 128 CTAS rows and BN columns of D. Warp 0 loads, warp 1
// multiplies, the others write results out.
template <int KIND, int BN, int CTAS>
struct Shape {
  static constexpr int kStoreWarps = KIND == WEIGHT_F32 ? 16 : 8;
  static constexpr int kRun = KIND == WEIGHT_F32 ? 768 : 4096;  // see "Precision" above
  static constexpr int kThreads = 64 + 32 * kStoreWarps;
  static constexpr int kStoreBytes = kStoreWarps * 32 * kStoreRow;
  static constexpr int kRows = kTileM * CTAS;
  static constexpr int kCols = BN / CTAS;  // columns of B that a CTA loads
  static constexpr int kStageBytes = (kTileM + kCols) * 128;
  static constexpr int kStages = (212992 - kStoreBytes) / kStageBytes;  // 3 to 8
  static constexpr int kTmemCols = 2 * BN;                              // two accumulators
  static constexpr int kBand = kBandRows / kRows;
  static constexpr int kSmem =
      1024 + kStages * kStageBytes + kStoreBytes + 8 * kGroupSlots + 512;
};

// Where piece `p` (16 bytes) of row `row` lies in a staging block: the 64-byte swizzle of TMA.
__device__ __forceinline__ uint32_t staged(int row, int p) {
  return row * kStoreRow + ((p ^ ((row >> 1) & 3)) << 4);
}

// One 32-row block of a storing warp, from its staging block to `dst` (row pitch in bytes),
// `bytes` of each row, UNIT bytes at a time.
template <int UNIT>
__device__ __forceinline__ void store_rows(uint32_t stage, char* dst, int64_t pitch, int nrows,
                                           int bytes, int lane) {
  constexpr int kLanes = kStoreRow / UNIT;  // of a row
  constexpr int kPerStep = 32 / kLanes;     // rows
  const int at = lane % kLanes * UNIT;
  if (at + UNIT > bytes) return;
  char* to = dst + (lane / kLanes) * pitch + at;
#pragma unroll 8
  for (int i0 = 0; i0 < 32; i0 += kPerStep) {
    const int i = i0 + lane / kLanes;
    if (i < nrows) {
      const uint32_t from = stage + staged(i, at >> 4) + (at & 15);
      if constexpr (UNIT == 16) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(from)
                     : "memory");
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
      } else if constexpr (UNIT == 8) {
        uint32_t w[2];
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                     : "=r"(w[0]), "=r"(w[1])
                     : "r"(from)
                     : "memory");
        *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
      } else if constexpr (UNIT == 4) {
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(from) : "memory");
        *reinterpret_cast<uint32_t*>(to) = w;
      } else {
        uint16_t w;
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(w) : "r"(from) : "memory");
        *reinterpret_cast<uint16_t*>(to) = w;
      }
    }
    to += kPerStep * pitch;
  }
}

struct Maps {
  CUtensorMap a, b;  // tiles of 64 columns
  CUtensorMap out;   // 32 rows of 64 bytes
};

template <int KIND, int BN, int CTAS>
__global__ void __launch_bounds__(Shape<KIND, BN, CTAS>::kThreads, 1)
    k_grouped_matmul(const __grid_constant__ Maps maps, const MatArgs g) {
  using S = Shape<KIND, BN, CTAS>;
  constexpr int MODE = KIND == WEIGHT_F32 ? (int)WEIGHT : KIND;
  constexpr int kLead = MODE == WEIGHT ? 0 : 1;  // groups before the first expert's
  constexpr bool kWide = KIND == WEIGHT_F32;  // results of 32 bits
  constexpr int kRun = S::kRun;
  constexpr int kStages = S::kStages;
  constexpr uint32_t kABytes = kTileM * 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t base = smem_addr(smem);
  const uint32_t store_base = base + kStages * S::kStageBytes;
  int32_t* cum = reinterpret_cast<int32_t*>(smem + kStages * S::kStageBytes + S::kStoreBytes);
  int32_t* off = cum + kGroupSlots;  // the groups' first rows, then the end
  uint64_t* bars = reinterpret_cast<uint64_t*>(
      (reinterpret_cast<uintptr_t>(off + kGroupSlots) + 15) & ~(uintptr_t)15);
  // end_full, end_peer (WEIGHT): a group's last block has landed in this CTA; the odd CTA has
  // zeroed its rows past the end. Used in turn, one a last block.
  const uint32_t full = smem_addr(bars), empty = full + 8 * kStages,
                 acc_full = empty + 8 * kStages, acc_empty = acc_full + 16,
                 end_full = acc_empty + 16, end_peer = end_full + 8 * kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 * kStages + 4);
  const int groups = g.experts + 2 * kLead;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? blockIdx.x & 1 : 0;  // in the pair; the even CTA multiplies

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        bar_init(full + 8 * i, 1);
        bar_init(empty + 8 * i, 1);
        bar_init(end_full + 8 * i, 1);
        bar_init(end_peer + 8 * i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        bar_init(acc_full + 8 * i, 1);
        bar_init(acc_empty + 8 * i, S::kStoreWarps * CTAS);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.b) : "memory");
    }
  } else if (warp == 1) {
    if constexpr (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_addr(tmem_slot)),
                   "r"((uint32_t)S::kTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_addr(tmem_slot)),
                   "r"((uint32_t)S::kTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  } else if (warp == 2) {
    // The groups' rows, clamped (off[i] to off[i + 1]; overlaps of offsets that decrease are
    // cut off), and the first tile of every group. The rows before the first offset are a group
    // of their own and so are those past the last; WEIGHT needs neither.
    const int nt = (g.cols + BN - 1) / BN;
    int32_t carry = 0, reach = 0;
    const int experts = MODE == WEIGHT ? g.experts / g.parts : g.experts;
    for (int i0 = 0; i0 <= experts; i0 += 32) {
      const int i = i0 + lane;
      int32_t b = i <= experts ? (int32_t)min(max((int64_t)g.offsets[i], (int64_t)0), g.rows) : 0;
      b = max(b, reach);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int32_t o = __shfl_up_sync(0xFFFFFFFFu, b, d);
        if (lane >= d) b = max(b, o);
      }
      reach = __shfl_sync(0xFFFFFFFFu, b, 31);
      if (i <= experts) off[kLead + i] = b;
    }
    if (MODE == WEIGHT && g.parts > 1) {  // each expert's rows in equal parts of whole blocks
      __syncwarp();
      for (int i = lane; i <= g.experts; i += 32) {
        const int e = i / g.parts, part = i % g.parts;
        const int32_t n = e < experts ? off[e + 1] - off[e] : 0;
        const int32_t each = part_rows(n, g.parts, kTileK);
        cum[i] = off[e] + (int32_t)min((int64_t)each * part, (int64_t)n);
      }
      __syncwarp();
      for (int i = lane; i <= g.experts; i += 32) off[i] = cum[i];
      __syncwarp();
    }
    if (kLead > 0 && lane == 0) {
      off[0] = 0;
      off[kLead + g.experts + 1] = (int32_t)g.rows;
    }
    __syncwarp();
    for (int i0 = 0; i0 < groups; i0 += 32) {
      const int i = i0 + lane;
      int32_t v = 0;
      if (i < groups)
        v = ((MODE == WEIGHT ? g.drows : off[i + 1] - off[i]) + S::kRows - 1) / S::kRows * nt;
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
  if constexpr (CTAS == 2) cluster_sync();  // the other CTA's barriers are set up too
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int tiles = cum[groups];
  const int nt = (g.cols + BN - 1) / BN;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  auto decode = [&](int t) {
    int lo = 0, hi = groups;  // the last group that starts at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] <= t) lo = mid; else hi = mid;
    }
    const int b = off[lo], e = off[lo + 1];
    Tile r;
    r.expert = lo - kLead;
    int m, n;
    const int drows = MODE == WEIGHT ? g.drows : e - b;
    tile_of(t - cum[lo], (drows + S::kRows - 1) / S::kRows, nt, S::kBand, m, n);
    r.n0 = n * BN;
    r.m0 = m * S::kRows + rank * kTileM;
    if (MODE == WEIGHT) {
      // Every group has the same tiles, the last row tile perhaps nearly empty: rotated by
      // group, so that a CTA does not meet the same one in each (their step through the tiles
      // is even).
      const int mt = (g.drows + S::kRows - 1) / S::kRows;
      m = (m + lo) % mt;
      r.m0 = m * S::kRows + rank * kTileM;
      r.m_end = g.drows;
      r.red0 = b;
      r.red = e - b;
    } else {
      r.m0 += b;
      r.m_end = e;
      r.red0 = 0;
      r.red = r.expert >= 0 && r.expert < g.experts ? g.reduction : 0;
    }
    return r;
  };

  // The half of tensor memory that run `run` of a tile goes to, and how often it was used before:
  // the multiplying and the storing warps count alike. WEIGHT_F32's runs alternate between the
  // halves; the others' tiles do, and their later runs all take the half that the first has not.
  uint32_t half = 1, used0 = 0, used1 = 0;
  auto take = [&](int run, uint32_t& acc) {
    if (kWide || run == 0) half ^= 1;
    acc = kWide || run == 0 ? half : half ^ 1;
    return acc ? used1++ : used0++;
  };

  bool ok = true;
  if (warp == 0) {
    uint32_t it = 0, ends = 0;
    for (int t = first; ok && t < tiles; t += step) {
      const Tile r = decode(t);
      const int nb = r.n0 + rank * S::kCols;  // first column of this CTA's share of B
      for (int k0 = 0; k0 < r.red; k0 += kTileK, ++it) {
        const uint32_t s = it % kStages;
        if (it >= kStages && !(ok = bar_wait(empty + 8 * s, (it / kStages - 1) & 1))) break;
        const uint32_t a = base + s * S::kStageBytes, b = a + kABytes;
        uint32_t bar = CTAS == 2 ? leader_addr(full + 8 * s) : full + 8 * s;
        const bool end = MODE == WEIGHT && r.red - k0 < kTileK;
        if (elect_one()) {
          if (end) {
            // lands at this CTA's own barrier; the stage's turns over without bytes
            bar = end_full + 8 * (ends % kStages);
            bar_expect(bar, S::kStageBytes);
            if (rank == 0) bar_expect(full + 8 * s, 0);
          } else if (rank == 0) {
            bar_expect(full + 8 * s, CTAS * S::kStageBytes);
          }
          if (MODE == WEIGHT) {
#pragma unroll
            for (int j = 0; j < kTileM / 64; ++j)
              tma_load_2d<CTAS>(a + j * 8192, &maps.a, r.m0 + 64 * j, r.red0 + k0, bar);
#pragma unroll
            for (int j = 0; j < S::kCols / 64; ++j)
              tma_load_2d<CTAS>(b + j * 8192, &maps.b, nb + 64 * j, r.red0 + k0, bar);
          } else {
            tma_load_2d<CTAS>(a, &maps.a, k0, r.m0, bar);
            if (MODE == FORWARD) {
              tma_load_3d<CTAS>(b, &maps.b, k0, nb, r.expert, bar);
            } else {
#pragma unroll
              for (int j = 0; j < S::kCols / 64; ++j)
                tma_load_3d<CTAS>(b + j * 8192, &maps.b, nb + 64 * j, k0, r.expert, bar);
            }
          }
        }
        __syncwarp();
        if (end) ++ends;
      }
    }
    // no copy may be in flight when the CTA ends: one whose block nobody multiplied (another
    // warp gave up, two seconds ago) has landed when these waits return or run out
    if (!ok) {
      for (uint32_t i = it > kStages ? it - kStages : 0; rank == 0 && i < it; ++i)
        bar_wait(full + 8 * (i % kStages), (i / kStages) & 1);
      if (ends > 0) bar_wait(end_full + 8 * ((ends - 1) % kStages), ((ends - 1) / kStages) & 1);
    }
  } else if (warp == 1) {
    uint32_t it = 0, ends = 0;
    for (int t = first; ok && t < tiles; t += step) {
      const Tile r = decode(t);
      uint32_t acc = 0, d = 0;
      for (int k0 = 0; k0 < r.red; k0 += kTileK, ++it) {
        const bool begin = k0 % kRun == 0;
        if (begin) {
          const uint32_t used = take(k0 / kRun, acc);
          d = tmem + acc * BN;
          if (rank == 0) {
            if (used > 0 && !(ok = bar_wait(acc_empty + 8 * acc, (used - 1) & 1))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
        }
        const uint32_t s = it % kStages;
        const uint32_t a = base + s * S::kStageBytes, b = a + kABytes;
        // the last block in whole steps of 16
        const int valid = min(r.red - k0, kTileK), steps = (valid + 15) / 16;
        const bool end = MODE == WEIGHT && valid < kTileK;
        if (end) {
          const uint32_t slot = 8 * (ends % kStages), parity = (ends / kStages) & 1;
          ++ends;
          if (!(ok = bar_wait(end_full + slot, parity))) break;
          const int rest = steps * 16 - valid;
          constexpr int kPanels = (kTileM + S::kCols) / 64;
          for (int i = lane; i < rest * kPanels * 8; i += 32) {
            const int panel = i / (rest * 8), row = i / 8 % rest;
            store_piece(a + panel * 8192 + (valid + row) * 128 + (i & 7) * 16, 0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (rank == 1) {
            if (lane == 0) bar_arrive_cluster(leader_addr(end_peer + slot));
          } else if (CTAS == 2 && !(ok = bar_wait(end_peer + slot, parity))) {
            break;
          }
        }
        const bool done = k0 + kTileK >= r.red || (k0 + kTileK) % kRun == 0;
        if (rank == 1) continue;  // the even CTA multiplies for both
        if (!(ok = bar_wait(full + 8 * s, (it / kStages) & 1))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_one()) {
          for (int k = 0; k < steps; ++k) {
            // 16 of the reduction: 32 bytes along a K-major row, 16 rows of an MN-major panel
            const uint64_t da = MODE == WEIGHT ? smem_desc(a + k * 2048, 8192, 1024)
                                               : smem_desc(a + k * 32, 16, 1024);
            const uint64_t db = MODE == FORWARD ? smem_desc(b + k * 32, 16, 1024)
                                                : smem_desc(b + k * 2048, 8192, 1024);
            mma_f16<CTAS>(d, da, db, g.idesc, !begin || k > 0);
          }
          mma_commit<CTAS>(empty + 8 * s);
          if (done) mma_commit<CTAS>(acc_full + 8 * acc);
        }
        __syncwarp();
      }
    }
  } else {
    const int quarter = warp & 3, part = (warp - 2) >> 2;  // of the lanes; of the chunks
    constexpr int kParts = S::kStoreWarps / 4;
    const uint32_t stage = store_base + (warp - 2) * 32 * kStoreRow;
    constexpr int bytes = kWide ? 4 : 2;
    constexpr int per_chunk = kStoreRow / bytes;  // columns of a staging row
    const int64_t pitch = g.out_pitch * bytes;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    auto accumulated = [&](int run, uint32_t& acc) {  // waits for that run
      const uint32_t used = take(run, acc);
      if (!bar_wait(acc_full + 8 * acc, used & 1)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return true;
    };
    auto release = [&](uint32_t acc) {  // this half has been read
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      const uint32_t bar = acc_empty + 8 * acc;
      if (lane == 0) bar_arrive_cluster(CTAS == 2 ? leader_addr(bar) : bar);
    };
    for (int t = first; ok && t < tiles; t += step) {
      const Tile r = decode(t);
      const int row0 = r.m0 + quarter * 32;
      char* out = static_cast<char*>(g.out);
      int out_row = row0;  // of D as one matrix
      if (MODE == WEIGHT) {
        out += (int64_t)r.expert * g.drows * pitch;
        out_row += r.expert * g.drows;
      }
      const int ncols = min(BN, g.cols - r.n0), nrows = min(32, r.m_end - row0);
      // whole 32-row blocks leave by TMA, which also cuts off the last columns
      const bool by_tma = g.unit == 16 && nrows == 32;
      // this lane's row of a chunk, 64 bytes, through the staging block to D
      auto put = [&](const uint32_t* w, int c0) {
        // the staging block is free when the last store has read it
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int p = 0; p < 4; ++p)
          store_piece(stage + staged(lane, p), w[4 * p], w[4 * p + 1], w[4 * p + 2],
                      w[4 * p + 3]);
        if (by_tma) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            asm volatile(
                "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                    &maps.out),
                "r"(r.n0 + c0), "r"(out_row), "r"(stage)
                : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          __syncwarp();
          const int n = min(per_chunk, ncols - c0) * bytes;
          char* dst = out + (int64_t)row0 * pitch + (int64_t)(r.n0 + c0) * bytes;
          if (g.unit == 16) store_rows<16>(stage, dst, pitch, nrows, n, lane);
          else if (g.unit == 8) store_rows<8>(stage, dst, pitch, nrows, n, lane);
          else if (g.unit == 4) store_rows<4>(stage, dst, pitch, nrows, n, lane);
          else store_rows<2>(stage, dst, pitch, nrows, n, lane);
        }
        __syncwarp();
      };
      uint32_t acc = 0;
      if (kWide && r.red > kRun) {
        constexpr int kMine = BN / per_chunk / kParts;  // chunks of this warp
        uint32_t sum[kMine][16];
#pragma unroll
        for (int i = 0; i < kMine; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) sum[i][j] = 0;
        for (int k0 = 0; k0 < r.red; k0 += kRun) {
          if (!(ok = accumulated(k0 / kRun, acc))) break;
          const uint32_t from = tmem + acc * BN + lanes + part * per_chunk;
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            uint32_t v[16];
            tmem_load16(from + i * kParts * per_chunk, v);
            tmem_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              sum[i][j] = __float_as_uint(__uint_as_float(sum[i][j]) + __uint_as_float(v[j]));
          }
          release(acc);
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if ((i * kParts + part) * per_chunk < ncols && nrows > 0)
            put(sum[i], (i * kParts + part) * per_chunk);
      } else {
        if (r.red > 0 && !(ok = accumulated(0, acc))) break;
        const uint32_t from = tmem + acc * BN + lanes;
        if constexpr (!kWide) {
          // each later run is added to the first one's half, where the sum leaves from
          for (int k0 = kRun; k0 < r.red; k0 += kRun) {
            uint32_t other;
            if (!(ok = accumulated(k0 / kRun, other))) break;
#pragma unroll 1
            for (int c0 = part * per_chunk; c0 < BN; c0 += kParts * per_chunk)
#pragma unroll 1
              for (int c = c0; c < c0 + per_chunk; c += 16) {
                uint32_t sum[16], v[16];
                tmem_load16(from + c, sum);
                tmem_load16(tmem + other * BN + lanes + c, v);
                tmem_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  sum[j] = __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(v[j]));
                tmem_store16(from + c, sum);
              }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            release(other);
          }
          if (!ok) break;
        }
        for (int c0 = part * per_chunk; c0 < ncols && nrows > 0; c0 += kParts * per_chunk) {
          uint32_t v[32], w[16];
          if (r.red == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = 0;
          } else if constexpr (kWide) {
            tmem_load16(from + c0, w);
            tmem_wait();
          } else {
            tmem_load32(from + c0, v);
            tmem_wait();
            if (g.out_kind == LGBM_B200_DTYPE_BF16) {
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = pack2<true>(v[2 * i], v[2 * i + 1]);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = pack2<false>(v[2 * i], v[2 * i + 1]);
            }
          }
          put(w, c0);
        }
        if (r.red > 0) release(acc);
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  if (!ok && lane == 0) atomicOr(g.error, 1u);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync();  // neither leaves while the other may still reach it
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) {
    if constexpr (CTAS == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"((uint32_t)S::kTmemCols));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"((uint32_t)S::kTmemCols));
  }
}

// Rows copied to a pitch that TMA can walk: dst[r] = src[index ? index[r] : r], the columns
// between `width` and `dst_pitch` zero; a row whose index is outside is zero.
// 2^LOG lanes a row and kRunOf pieces of 16 bytes a lane at a time, all loads first: a warp a
// row and four pieces from 512 bytes on, half as many lanes as pieces for short rows. UNIT is
// the rows' alignment, 2 for all below 8. Measured, rows x columns: 40009 x 700 (8 bytes) 18 us,
// 6.1 TB/s read and written; 65536 x 2755 110 us, 6.6; 7884 x 3977 25 us, 5.0; 40009 x 129 6.9
// us (a warp a row 10.7), 500000 x 21 10 us (a warp a row and 2 bytes a load: 44 for 556780).
constexpr int kStageRun = 4;

// `left`: bytes of the row from p on.
template <int UNIT>
__device__ __forceinline__ uint4 stage_piece(const char* p, int left) {
  if (UNIT == 16 && left >= 16) return __ldg(reinterpret_cast<const uint4*>(p));
  if (UNIT >= 8 && left >= 16) {
    const uint2 lo = __ldg(reinterpret_cast<const uint2*>(p));
    const uint2 hi = __ldg(reinterpret_cast<const uint2*>(p + 8));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  uint32_t e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    e[j] = 2 * j < left ? __ldg(reinterpret_cast<const uint16_t*>(p) + j) : 0;
  return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}

// The same from any even address: the one or two aligned pieces that hold it, loaded by
// stage_load, shifted here. (Eight loads of 2 bytes a piece pass through L1 one by one.)
struct StagePair { uint4 a, b; };
__device__ __forceinline__ StagePair stage_load(const char* p, int left) {
  const int s = (int)(reinterpret_cast<uintptr_t>(p) & 15);
  const uint4* q = reinterpret_cast<const uint4*>(p - s);
  return {__ldg(q), __ldg(q + (s + min(left, 16) > 16))};
}
__device__ __forceinline__ uint4 stage_shift(const StagePair& v, int s, int left) {
  uint32_t w[8] = {v.a.x, v.a.y, v.a.z, v.a.w, v.b.x, v.b.y, v.b.z, v.b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = s & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = s & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = s & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
  if (left < 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = left >= 4 * i + 4 ? w[i] : left > 4 * i ? w[i] & 0xFFFFu : 0;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int UNIT, int LOG>
__global__ void __launch_bounds__(256)
    k_stage_rows(const char* __restrict__ src, int64_t src_rows, int64_t rows, int bytes,
                 int64_t pitch, const int32_t* __restrict__ index, char* __restrict__ dst,
                 int dst_bytes) {
  constexpr int kLanes = 1 << LOG, kRunOf = LOG == 5 ? kStageRun : 2, kStep = 16 * kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t r = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (r >= rows) return;
  const int64_t at = index ? index[r] : r;
  const bool inside = at >= 0 && at < src_rows;
  const char* from = src + (inside ? at : 0) * pitch;
  char* to = dst + r * dst_bytes;
  if constexpr (UNIT < 8) {
    // aligned pieces may begin before a row and end behind it, but not outside the source
    const int s = (int)(reinterpret_cast<uintptr_t>(from) & 15);
    const int64_t behind = src + (src_rows - 1) * pitch - from;  // this row's end to the last's
    if (inside && from - s >= src && (-(s + bytes) & 15) <= behind) {
      for (int c0 = lane * 16; c0 < dst_bytes; c0 += kStep * kRunOf) {
        StagePair v[kRunOf];
#pragma unroll
        for (int u = 0; u < kRunOf; ++u) {
          const int c = c0 + kStep * u;
          v[u] = c < bytes ? stage_load(from + c, bytes - c) : StagePair();
        }
#pragma unroll
        for (int u = 0; u < kRunOf; ++u) {
          const int c = c0 + kStep * u;
          if (c < dst_bytes)
            *reinterpret_cast<uint4*>(to + c) = stage_shift(v[u], s, bytes - c);
        }
      }
      return;
    }
  }
  for (int c0 = lane * 16; c0 < dst_bytes; c0 += kStep * kRunOf) {
    uint4 v[kRunOf];
#pragma unroll
    for (int u = 0; u < kRunOf; ++u) {
      const int c = c0 + kStep * u;
      v[u] = make_uint4(0, 0, 0, 0);
      if (inside && c < bytes) v[u] = stage_piece<UNIT>(from + c, bytes - c);
    }
#pragma unroll
    for (int u = 0; u < kRunOf; ++u)
      if (c0 + kStep * u < dst_bytes) *reinterpret_cast<uint4*>(to + c0 + kStep * u) = v[u];
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

// A tensor, innermost axis first; boxes of `row` bytes (64 or 128, swizzled alike) x `box1`
// rows, zeros outside the tensor.
bool encode(CUtensorMap* map, int32_t dtype, const void* base, int rank, const int64_t* dims,
            const int64_t* pitches, int box1, int row = 128) {
  const int bytes = elem_size(dtype);
  cuuint64_t d[3], s[2];
  cuuint32_t box[3] = {(cuuint32_t)(row / bytes), (cuuint32_t)box1, 1}, step[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) d[i] = (cuuint64_t)dims[i];
  for (int i = 0; i + 1 < rank; ++i) s[i] = (cuuint64_t)pitches[i] * bytes;
  const EncodeTiled fn = encoder();
  return fn && fn(map,
                  dtype == LGBM_B200_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                  : dtype == LGBM_B200_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  (cuuint32_t)rank, const_cast<void*>(base), d, s, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE,
                  row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a launch needs to know of the current device, looked up once a device.
constexpr int kMaxDevices = 64;
struct DeviceInfo {
  std::mutex mu;
  uint32_t* error = nullptr;
};
DeviceInfo g_devices[kMaxDevices];

template <int KIND, int BN, int CTAS>
cudaError_t launch_tiles(const Maps& maps, MatArgs g, int64_t most_tiles, cudaStream_t st) {
  using S = Shape<KIND, BN, CTAS>;
  static std::atomic<int> most_ready[kMaxDevices];  // tiles at work at a time; 0: not set up
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  {
    DeviceInfo& d = g_devices[dev];
    std::lock_guard<std::mutex> lock(d.mu);
    if (!d.error) {
      void* p = nullptr;
      err = cudaGetSymbolAddress(&p, g_matmul_error);
      if (err != cudaSuccess) return err;
      d.error = static_cast<uint32_t*>(p);
    }
    g.error = d.error;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(CTAS, 1, 1);
  cfg.blockDim = dim3(S::kThreads, 1, 1);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CTAS;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CTAS == 2 ? 1 : 0;
  int most = most_ready[dev].load(std::memory_order_acquire);
  if (most == 0) {
    err = cudaFuncSetAttribute(k_grouped_matmul<KIND, BN, CTAS>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    // a pair that finds no room would start when the others have finished: ask how many fit
    if (err == cudaSuccess && CTAS == 2)
      err = cudaOccupancyMaxActiveClusters(&most, k_grouped_matmul<KIND, BN, CTAS>, &cfg);
    else if (err == cudaSuccess)
      err = cudaDeviceGetAttribute(&most, cudaDevAttrMultiProcessorCount, dev);
    if (err != cudaSuccess) return err;
    if (most < 1) return cudaErrorInvalidConfiguration;
    most_ready[dev].store(most, std::memory_order_release);
  }
  cfg.gridDim.x = (unsigned)(std::min<int64_t>(most, most_tiles) * CTAS);
  return cudaLaunchKernelEx(&cfg, k_grouped_matmul<KIND, BN, CTAS>, maps, g);
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
  char* dst = workspace;
  workspace += copy_bytes(rows, width);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(o.p) | (uintptr_t)(o.pitch * 2);
  auto go = [&](auto unit, auto log) {
    constexpr int kRows = 256 >> decltype(log)::value;
    const int64_t blocks = (rows + kRows - 1) / kRows;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    k_stage_rows<decltype(unit)::value, decltype(log)::value><<<(unsigned)blocks, 256, 0, st>>>(
        static_cast<const char*>(o.p), src_rows, rows, width * 2, o.pitch * 2, index, dst,
        (int)(dst_pitch * 2));
    return cudaGetLastError();
  };
  auto with_lanes = [&](auto unit) {
    if (dst_pitch <= 32) return go(unit, std::integral_constant<int, 1>());
    if (dst_pitch <= 128) return go(unit, std::integral_constant<int, 3>());
    if (dst_pitch <= 256) return go(unit, std::integral_constant<int, 4>());
    return go(unit, std::integral_constant<int, 5>());
  };
  const cudaError_t err = bits % 16 == 0  ? with_lanes(std::integral_constant<int, 16>())
                          : bits % 8 == 0 ? with_lanes(std::integral_constant<int, 8>())
                                          : with_lanes(std::integral_constant<int, 2>());
  o.p = dst;
  o.pitch = dst_pitch;
  return err;
}

uint32_t instruction(int32_t dtype, bool a_mn, bool b_mn, int m, int n) {
  const uint32_t type = dtype == LGBM_B200_DTYPE_BF16 ? 1 : 0;
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn << 15) |
         ((uint32_t)b_mn << 16) | ((uint32_t)(n / 8) << 17) | ((uint32_t)(m / 16) << 24);
}

// Whether an expert's weight gradient of more than 128 columns is multiplied by pairs.
bool weight_pairs(int64_t drows) { return drows >= kTileM * 3 / 2; }

// a: x (FORWARD) or dy; b: w, or x (WEIGHT).
template <int MODE>
cudaError_t run_tiles(const Operand& a, int64_t a_width, const Operand& b, int64_t b_width,
                      int32_t dtype, MatArgs g, cudaStream_t st) {
  const int bytes = elem_size(g.out_kind);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(g.out) | (uintptr_t)(g.out_pitch * bytes) |
                         (uintptr_t)(g.cols * bytes);
  g.unit = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
  auto go = [&](auto bn_c, auto ctas_c) -> cudaError_t {
    constexpr int BN = decltype(bn_c)::value, CTAS = decltype(ctas_c)::value;
    using S = Shape<MODE, BN, CTAS>;
    Maps maps;
    const int64_t da[3] = {a_width, g.rows, 1}, pa[2] = {a.pitch, 0};
    bool fine = encode(&maps.a, dtype, a.p, 2, da, pa, MODE == WEIGHT ? 64 : kTileM);
    if (MODE == WEIGHT) {
      const int64_t db[3] = {b_width, g.rows, 1}, pb[2] = {b.pitch, 0};
      fine = fine && encode(&maps.b, dtype, b.p, 2, db, pb, 64);
    } else {
      const int64_t n = MODE == FORWARD ? g.cols : g.reduction;
      const int64_t db[3] = {b_width, n, g.experts}, pb[2] = {b.pitch, b.pitch * n};
      fine = fine && encode(&maps.b, dtype, b.p, 3, db, pb, MODE == FORWARD ? S::kCols : 64);
    }
    maps.out = maps.a;  // not used unless set
    const int64_t rows_d = MODE == WEIGHT ? (int64_t)g.experts * g.drows : g.rows;
    if (g.unit == 16 && rows_d > INT32_MAX) g.unit = 8;  // no coordinate for its last rows
    if (g.unit == 16) {
      const int64_t dd[3] = {g.cols, rows_d, 1}, pd[2] = {g.out_pitch, 0};
      fine = fine && encode(&maps.out, g.out_kind, g.out, 2, dd, pd, 32, kStoreRow);
    }
    if (!fine) return cudaErrorInvalidValue;
    g.idesc = instruction(dtype, MODE == WEIGHT, MODE != FORWARD, S::kRows, BN);
    const int64_t nt = (g.cols + BN - 1) / BN;
    const int64_t most = MODE == WEIGHT
                             ? (int64_t)g.experts * ((g.drows + S::kRows - 1) / S::kRows) * nt
                             : (g.rows / S::kRows + g.experts + 2) * nt;
    if (MODE == WEIGHT && g.out_kind == LGBM_B200_DTYPE_F32)
      return launch_tiles<WEIGHT_F32, BN, CTAS>(maps, g, most, st);
    return launch_tiles<MODE, BN, CTAS>(maps, g, most, st);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (g.cols <= 64) return go(std::integral_constant<int, 64>(), One());
  if (g.cols <= 128) return go(std::integral_constant<int, 128>(), One());
  // Pairs where most tiles fill more than one and a half CTAs' rows, or an expert's rows more
  // than one's: else the odd CTA of a pair has little to do. (255 experts of 136 x 704 with 157
  // rows on average: y 33 us either way; dw in f32 67 in pairs, 59 without.)
  const bool tall = MODE == WEIGHT ? weight_pairs(g.drows) : g.rows >= (int64_t)kTileM * g.experts;
  return tall ? go(std::integral_constant<int, 256>(), Two())
              : go(std::integral_constant<int, 256>(), One());
}

// Sums of the parts of a weight gradient, always in the same order: part[e][p][n] to out[e][n],
// n in [0, count). V elements a thread.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    k_join_parts(const float* part, int parts, int64_t count, int64_t total, T* out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= total) return;
  const int64_t e = i / count;
  const float* p = part + e * count * (parts - 1) + i;  // (e * parts) * count + i - e * count
  float sum[V] = {};
#pragma unroll 4
  for (int k = 0; k < parts; ++k, p += count) {
    if constexpr (V == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
    } else {
      sum[0] += *p;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) out[i + j] = from_f32<T>(sum[j]);
}

template <typename T>
cudaError_t join_parts(const float* part, int parts, int64_t count, int experts, T* out,
                       cudaStream_t st) {
  const int64_t total = count * experts;
  const auto blocks = [&](int v) { return (unsigned)((total / v + 255) / 256); };
  if (count % 4 == 0)
    k_join_parts<T, 4><<<blocks(4), 256, 0, st>>>(part, parts, count, total, out);
  else
    k_join_parts<T, 1><<<blocks(1), 256, 0, st>>>(part, parts, count, total, out);
  return cudaGetLastError();
}

}  // namespace

// Whether the forward product streams its weights (experts_few.cu) instead of multiplying
// tiles. Measured, streamed / tiles in us, weights from memory, at rows an expert (all with rows):
// - Weights that TMA walks: up to 2 rows it saves the tiles' longer start (8 experts of 4096 x
//   2048: 2 rows 28.8 / 35.1, 4 28.9 / 28.9, 8 30.2 / 29.0). Few tiles leave SMs idle, while
//   streaming splits the inner axis: up to 32 rows (2 of 512 x 512: 8.5 / 10.3).
// - Others would be copied first, all experts' even where few have rows. Small weights: the
//   copy's launch and latency cost more than streaming up to 32 rows (64 of 128 x 129: 10.5 /
//   16.5; 64 of 256 x 257: 14.5 / 22.7).
// - Rows at 4 bytes: to about 24 (32 of 4096 x 2002: 24 rows 253 / 269, 32 289 / 271), fewer where
//   the last block of 128 outputs is mostly empty (255 of 129 x 700: 8 rows 41.4 / 42.3, 12 47.4
//   / 44.1, 24 57.0 / 45.4).
// - Rows at 2 bytes: they come by 2-byte loads, each waited for. Streaming pays while it leaves
//   out half of the experts (32 of 4096 x 2001: rows of 16 experts 198 / 234, of 20 287 / 240, of
//   32 383 / 295; 8 of 4096 x 4097: of 4 109 / 149, of 5 183 / 161).
constexpr int64_t kSmallWeights = 12 << 20;
static bool few_rows(const MatmulCall& c) {
  if (!c.y || c.rows > 32 * (int64_t)c.experts) return false;
  const int64_t outputs = (int64_t)c.experts * c.outer;
  if (aligned16(c.w) && c.inner % 8 == 0)
    return c.rows <= 2 * (int64_t)c.experts ||
           (int64_t)c.experts * ((c.outer + 255) / 256) < 148 / 2;
  if (outputs <= kSmallWeights / 2 / c.inner) return true;
  if (reinterpret_cast<uintptr_t>(c.w) % 4 == 0 && c.inner % 2 == 0)
    return c.rows * ((c.outer + 127) / 128 * 128) <= 24 * outputs;
  return 2 * c.rows <= c.experts;
}
static bool copies_x(const MatmulCall& c) {
  return ((c.y && !few_rows(c)) || c.dw) && (c.index || !walkable(c.x, c.x_pitch));
}
static bool copies_dy(const MatmulCall& c) {
  return (c.dx || c.dw) && !walkable(c.dy, c.dy_pitch);
}
static bool copies_w(const MatmulCall& c) {
  return ((c.y && !few_rows(c)) || c.dx) && !(aligned16(c.w) && c.inner % 8 == 0);
}

// Parts of each expert's rows that a weight gradient is summed in, 1: not split. Its tiles are
// its outputs', so few and small experts leave SMs idle while others walk all rows. Parts give
// every SM a tile; each has 256 rows on average at least, since a tile's start and end cost
// about that much and each part is written and read once in f32. Measured with the joining,
// without parts: 60330 rows, 3 experts of 80 x 2864 in f32 82, 183 us; 35996 rows, 19 of 56 x 80
// in bf16 18, 51; 1514 rows, 2 of 128 x 320 15.4, 17.4.
static int weight_parts(const MatmulCall& c) {
  const bool pairs = c.inner > 128 && weight_pairs(c.outer);
  const int64_t bn = c.inner <= 64 ? 64 : c.inner <= 128 ? 128 : 256;
  const int64_t tile_rows = pairs ? 2 * kTileM : kTileM;
  const int64_t tiles =
      c.experts * ((c.outer + tile_rows - 1) / tile_rows) * ((c.inner + bn - 1) / bn);
  const int64_t parts = std::min({(pairs ? 74 : 148) / tiles, c.rows / (256 * (int64_t)c.experts),
                                  (int64_t)(kMaxExperts / c.experts)});
  return c.dw && parts > 1 ? (int)parts : 1;
}
static int64_t parts_bytes(const MatmulCall& c) {
  const int parts = weight_parts(c);
  return parts > 1 ? sizeof(float) * parts * c.experts * (int64_t)c.outer * c.inner : 0;
}

int64_t matmul_workspace(const MatmulCall& c) {
  return parts_bytes(c) + (copies_x(c) ? copy_bytes(c.rows, c.inner) : 0) +
         (copies_dy(c) ? copy_bytes(c.rows, c.outer) : 0) +
         (copies_w(c) ? copy_bytes((int64_t)c.experts * c.outer, c.inner) : 0);
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
    f.y = c.y;
    return launch_few(f, st);
  }
  char* ws = static_cast<char*>(workspace);
  Operand x{c.x, c.x_pitch}, dy{c.dy, c.dy_pitch}, w{c.w, c.inner};
  cudaError_t err = cudaSuccess;
  if (copies_x(c)) err = stage(x, c.x_rows, c.rows, c.inner, c.index, ws, st);
  if (err == cudaSuccess && copies_dy(c))
    err = stage(dy, c.rows, c.rows, c.outer, nullptr, ws, st);
  const int64_t w_rows = (int64_t)c.experts * c.outer;
  if (err == cudaSuccess && copies_w(c))
    err = stage(w, w_rows, w_rows, c.inner, nullptr, ws, st);
  MatArgs g{};
  g.offsets = c.offsets;
  g.experts = c.experts;
  g.parts = 1;
  g.rows = c.rows;
  if (err == cudaSuccess && c.y) {
    g.out = c.y;
    g.out_kind = c.dtype;
    g.cols = c.outer;
    g.reduction = c.inner;
    g.out_pitch = c.outer;
    err = run_tiles<FORWARD>(x, c.inner, w, c.inner, c.dtype, g, st);
  }
  if (err == cudaSuccess && c.dx) {
    g.out = c.dx;
    g.out_kind = c.dtype;
    g.cols = c.inner;
    g.reduction = c.outer;
    g.out_pitch = c.inner;
    err = run_tiles<INPUT>(dy, c.outer, w, c.inner, c.dtype, g, st);
  }
  if (err == cudaSuccess && c.dw) {
    g.parts = weight_parts(c);
    g.experts *= g.parts;
    g.out = g.parts > 1 ? ws : c.dw;  // ws: the end of the copies
    g.out_kind = g.parts > 1 ? (int32_t)LGBM_B200_DTYPE_F32 : c.grad_dtype;
    g.cols = c.inner;
    g.drows = c.outer;
    g.out_pitch = c.inner;
    err = run_tiles<WEIGHT>(dy, c.outer, x, c.inner, c.dtype, g, st);
    if (err == cudaSuccess && g.parts > 1) {
      const int64_t count = (int64_t)c.outer * c.inner;
      const float* part = reinterpret_cast<const float*>(ws);
      if (c.grad_dtype == LGBM_B200_DTYPE_F32)
        err = join_parts(part, g.parts, count, c.experts, static_cast<float*>(c.dw), st);
      else if (c.grad_dtype == LGBM_B200_DTYPE_BF16)
        err = join_parts(part, g.parts, count, c.experts, static_cast<__nv_bfloat16*>(c.dw), st);
      else
        err = join_parts(part, g.parts, count, c.experts, static_cast<__half*>(c.dw), st);
    }
  }
  return err;
}

// Moves the error bits to where no kernel sets any, in one step: a bit that another thread's
// kernel sets meanwhile is in this answer or in the next.
static __device__ uint32_t g_taken_error;
static __global__ void k_take_errors() { g_taken_error = atomicExch(&g_matmul_error, 0u); }

// Waits for the whole device: work on streams that do not order with the legacy default stream,
// as those of torch's pool, would go unnoticed otherwise.
cudaError_t take_matmul_errors(uint32_t* bits) {
  static std::mutex mu;  // g_taken_error is one word a device
  cudaError_t err = cudaDeviceSynchronize();
  if (err != cudaSuccess) return err;
  std::lock_guard<std::mutex> lock(mu);
  k_take_errors<<<1, 1>>>();
  err = cudaGetLastError();
  return err != cudaSuccess ? err : cudaMemcpyFromSymbol(bits, g_taken_error, sizeof(*bits));
}

}  // namespace experts
}  // namespace lgbm_b200
