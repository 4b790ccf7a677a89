// Routing rows to experts: the k largest logits of every row with their softmax weights, and
// the rows' places when grouped by expert; the gradient of the weights.
#include "experts.cuh"

namespace lgbm_b200 {
namespace experts {
namespace {

constexpr int kRouteThreads = 256;   // k_route_place
constexpr uint32_t kKeyEmpty = 0x007FFFFFu;  // key of -inf: never chosen

// Order-preserving key of a logit: larger logit, larger key; -0 and +0 are one value, NaN
// ranks above everything (it is then chosen, and its row's weights are NaN).
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return v != v ? 0xFFFFFFFFu : key;
}
__device__ __forceinline__ float key_logit(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// Stable places of a block's slots, in slot order. chosen(i) gives slot i's expert (-1:
// none); base[e] is the first place of the block's rows of expert e (e = experts: the slots
// without an expert). Each warp ranks a contiguous run of slots: among 32 slots by matching
// lanes, across its runs by a counter per expert that only it writes.
template <int THREADS, typename Chosen>
__device__ void place_slots(int slots, int64_t first_slot, int experts, int k,
                            const Chosen& chosen, int32_t* base, int32_t* hist,
                            int32_t* position, int32_t* rows) {
  constexpr int kWarps = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = experts + 1;
  for (int i = threadIdx.x; i < kWarps * groups; i += THREADS) hist[i] = 0;
  __syncthreads();
  const int per_warp = ((slots + THREADS - 1) / THREADS) * 32;
  const int begin = warp * per_warp;
  int32_t* mine = hist + warp * groups;
  for (int i0 = begin; i0 < begin + per_warp && i0 < slots; i0 += 32) {
    const int i = i0 + lane;
    int e = -2;
    if (i < slots) {
      e = chosen(i);
      if (e < 0) e = experts;
    }
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    if (e >= 0 && (same & ((1u << lane) - 1u)) == 0) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < groups; e += THREADS) {
    int32_t at = base[e];
    for (int w = 0; w < kWarps; ++w) {
      const int32_t n = hist[w * groups + e];
      hist[w * groups + e] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int i0 = begin; i0 < begin + per_warp && i0 < slots; i0 += 32) {
    const int i = i0 + lane;
    int e = -2;
    if (i < slots) {
      e = chosen(i);
      if (e < 0) e = experts;
    }
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    const uint32_t before = same & ((1u << lane) - 1u);
    int32_t at = 0;
    if (e >= 0) at = mine[e];
    __syncwarp();
    if (e >= 0) {
      if (before == 0) mine[e] = at + __popc(same);
      at += __popc(before);
      position[first_slot + i] = at;
      rows[at] = (int32_t)((first_slot + i) / k);
    }
    __syncwarp();
  }
}

// Exclusive prefix of n <= kMaxExperts + 1 counts in shared memory by the first warp.
__device__ void prefix_counts(int32_t* counts, int n) {
  if (threadIdx.x < 32) {
    int32_t carry = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + threadIdx.x;
      const int32_t v = i < n ? counts[i] : 0;
      int32_t s = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int32_t o = __shfl_up_sync(0xFFFFFFFFu, s, d);
        if ((int)threadIdx.x >= d) s += o;
      }
      if (i < n) counts[i] = carry + s - v;
      carry += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// e^x for a term of a softmax's sum, x <= 0, in two instructions (with expf routing 65521 x 255
// takes 55.4 us instead of 51.6). The product is rounded, so a term is off by (|x| + 4) 2^-24 of
// itself. In the sum that is at most (ln E + 4) 2^-24 of the whole, 10 units for 512 experts,
// since the mean of |x| under the softmax is its entropy less ln of the sum. A result that is a
// single term takes expf.
__device__ __forceinline__ float exp_term(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

struct Choice {
  int id;            // an expert, -1: none left
  float own, total;  // weight: own / total
  __device__ __forceinline__ float weight() const { return id >= 0 ? own / total : 0.0f; }
};

// One token's choice by a warp, the j-th in lane j: expert i * 32 + lane is v[i], -inf where there
// is none. Searching all registers once a choice
// is what would cost most, so with CN < NV the choice has two stages: the k lanes with the
// largest maxima (ties to the lower expert) hold the k largest logits among them, since each lane
// left out has k elements before all of its own; their k * NV logits are dealt out to the 32
// lanes, CN each, and the k choices are made there, each one a maximum over the warp, the first
// expert that holds it, and its removal. Keys order as the logits do, with NaN above everything.
// The weights' bits depend on the token alone, not on NV, CN or the batch.
template <int NV, int CN>
__device__ __forceinline__ Choice choose(const float (&v)[NV], int k, bool normalize) {
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  constexpr bool kTwoStages = CN < NV;
  const int lane = threadIdx.x & 31;
  const float kNone = -__int_as_float(0x7F800000);
  float top = v[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) top = max_nan(top, v[i]);

  uint32_t key[CN];
  int id[CN];  // expert of a candidate
  if constexpr (kTwoStages) {
    // this lane's first register that holds its maximum (NaN: the first NaN)
    int at = 0;
#pragma unroll
    for (int i = NV - 1; i >= 0; --i)
      if (v[i] == top) at = i;
    if (top != top) {
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (v[i] != v[i]) at = i;
    }
    uint32_t lane_key = logit_key(top);
    int from[CN];  // lane that this lane's candidates come from: number (32 c + lane) / NV
#pragma unroll
    for (int c = 0; c < CN; ++c) from[c] = -1;
    for (int j = 0; j < k; ++j) {
      const uint32_t best = __reduce_max_sync(kAll, lane_key);
      if (best == kKeyEmpty) break;
      const int owner = (int)(__reduce_min_sync(kAll, lane_key == best
                                                          ? (uint32_t)(at * 32 + lane)
                                                          : kAll) & 31);
      if (lane == owner) lane_key = kKeyEmpty;
#pragma unroll
      for (int c = 0; c < CN; ++c)
        if ((c * 32 + lane) / NV == j) from[c] = owner;
    }
    // candidate lane % NV of each lane's source
#pragma unroll
    for (int c = 0; c < CN; ++c) {
      float x = kNone;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float y = __shfl_sync(kAll, v[i], from[c] & 31);
        if (lane % NV == i) x = y;
      }
      key[c] = from[c] < 0 ? kKeyEmpty : logit_key(x);
      id[c] = key[c] == kKeyEmpty ? 0 : (lane % NV) * 32 + from[c];
    }
  } else {
#pragma unroll
    for (int c = 0; c < CN; ++c) {
      key[c] = logit_key(v[c]);
      id[c] = c * 32 + lane;
    }
  }

  uint32_t my_key = kKeyEmpty;
  int my_id = -1;
  float m = 0.0f;
  for (int j = 0; j < k; ++j) {
    uint32_t mine = key[0];
#pragma unroll
    for (int c = 1; c < CN; ++c) mine = max(mine, key[c]);
    const uint32_t best = __reduce_max_sync(kAll, mine);
    if (best == kKeyEmpty) break;  // the same in every lane
    if (j == 0) m = key_logit(best);
    uint32_t e = kAll;
#pragma unroll
    for (int c = 0; c < CN; ++c)
      if (key[c] == best) e = min(e, (uint32_t)id[c]);
    e = __reduce_min_sync(kAll, e);
#pragma unroll
    for (int c = 0; c < CN; ++c)
      if ((uint32_t)id[c] == e) key[c] = kKeyEmpty;
    if (lane == j) {
      my_key = best;
      my_id = (int)e;
    }
  }
  const float mine = my_id >= 0 ? expf(key_logit(my_key) - m) : 0.0f;
  float total = mine;
  if (!normalize) {
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) total += exp_term(v[i] - m);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(kAll, total, d);
  return {my_id, mine, total};
}

constexpr int kSelectThreads = 256;
// Tokens of a block: a warp takes 1 to 16 of them, one after the other. One costs about 1.5 us,
// most of it the waits of its own choices, so few tokens are spread over up to 256 blocks
// before a warp takes more (109 rows of 199, k 6: 3.4 us, in blocks of 128 25; 1167 of 330: 3.8
// and 30); 16 a warp keep the counts, a number a block and expert, below the logits' bytes.
int select_tokens_of(int64_t tokens) {
  int n = kSelectThreads / 32;
  while (n < kSelectThreads / 2 && (tokens + n - 1) / n > 256) n *= 2;
  return n;
}

// First of three launches for many tokens: choice and weights, and each block's rows per
// expert. A warp a token, its logits in registers; the next token's are on their way meanwhile.
// Bound by instructions: 65521 rows of 255 f32 logits, k 4, take 41 us (67 MB: 1.6 TB/s) with
// 438 instructions a row and three quarters of the issue slots used. A sorted list a thread
// in registers took 71 us, a search of all registers a choice 64.
template <typename T, int NV, int CN>
__global__ void __launch_bounds__(kSelectThreads)
    k_route_select(const T* logits, int64_t tokens, int experts, int64_t pitch, int k,
                   bool normalize, int block_tokens, float* weights, int32_t* chosen,
                   int32_t* counts) {
  constexpr int kWarps = kSelectThreads / 32;
  __shared__ int32_t hist[kMaxExperts + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i <= experts; i += kSelectThreads) hist[i] = 0;
  __syncthreads();
  const int per_warp = block_tokens / kWarps;
  const int64_t first = (int64_t)blockIdx.x * block_tokens + warp * per_warp;
  const int64_t last = min(first + per_warp, tokens);
  const float kNone = -__int_as_float(0x7F800000);
  float next[NV];
  auto fetch = [&](const T* row) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      next[i] = i * 32 + lane < experts ? to_f32<T>(row[i * 32 + lane]) : kNone;
  };
  if (first < last) fetch(logits + first * pitch);
  for (int64_t t = first; t < last; ++t) {
    float v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = next[i];
    if (t + 1 < last) fetch(logits + (t + 1) * pitch);
    const Choice c = choose<NV, CN>(v, k, normalize);
    if (lane < k) {
      weights[t * k + lane] = c.weight();
      chosen[t * k + lane] = c.id;
      atomicAdd(&hist[c.id < 0 ? experts : c.id], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kSelectThreads)
    counts[(int64_t)e * gridDim.x + blockIdx.x] = hist[e];
}

// Second: per expert, the exclusive prefix of the blocks' counts; one warp an expert.
__global__ void __launch_bounds__(256) k_route_scan(int32_t* counts, int32_t* totals, int groups,
                                                    int blocks) {
  const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= groups) return;
  int32_t* row = counts + (int64_t)e * blocks;
  int32_t carry = 0;
  for (int i0 = 0; i0 < blocks; i0 += 32) {
    const int i = i0 + lane;
    const int32_t v = i < blocks ? row[i] : 0;
    int32_t s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int32_t o = __shfl_up_sync(0xFFFFFFFFu, s, d);
      if (lane >= d) s += o;
    }
    if (i < blocks) row[i] = carry + s - v;
    carry += __shfl_sync(0xFFFFFFFFu, s, 31);
  }
  if (lane == 0) totals[e] = carry;
}

// Third: offsets, and every slot's place. 7 us at 262084 slots and 255 experts (the scan 3):
// latency, not bandwidth; its 2 MB of results go to 255 ranges.
__global__ void __launch_bounds__(kRouteThreads)
    k_route_place(const int32_t* chosen, const int32_t* counts, const int32_t* totals,
                  int64_t tokens, int experts, int k, int block_tokens, int32_t* position,
                  int32_t* rows, int32_t* offsets) {
  extern __shared__ int32_t smem[];
  int32_t* base = smem;
  int32_t* hist = smem + experts + 1;
  for (int e = threadIdx.x; e <= experts; e += kRouteThreads) base[e] = totals[e];
  __syncthreads();
  prefix_counts(base, experts + 1);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= experts; e += kRouteThreads) offsets[e] = base[e];
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kRouteThreads)
    base[e] += counts[(int64_t)e * gridDim.x + blockIdx.x];
  const int64_t first = (int64_t)blockIdx.x * block_tokens;
  const int n = (int)min((int64_t)block_tokens, tokens - first) * k;
  const int32_t* mine = chosen + first * k;
  place_slots<kRouteThreads>(
      n, first * k, experts, k, [&](int i) { return mine[i]; }, base, hist, position, rows);
}

// A few tokens: all of it in one block and one launch, a warp a token. One row of 8 experts: 2.9
// us, of which the launch is most; 64 rows of 64, k 2, 6.5; 64 of 255, k 4, 9.8. (Three launches
// take 8.7 at 109 rows of 199, k 6.)
constexpr int kSmallThreads = 512;
constexpr int kSmallTokens = 64;  // most tokens this path takes: four a warp

template <typename T, int NV>
__global__ void __launch_bounds__(kSmallThreads)
    k_route_small(const T* logits, int tokens, int experts, int64_t pitch, int k,
                  bool normalize, float* weights, int32_t* chosen, int32_t* position,
                  int32_t* rows, int32_t* offsets) {
  extern __shared__ int32_t smem[];
  int32_t* ids = smem;                                 // kSmallTokens * k
  int32_t* base = ids + kSmallTokens * kMaxChosen;     // experts + 1
  int32_t* hist = base + experts + 1;                  // warps * (experts + 1)
  const int lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e <= experts; e += kSmallThreads) base[e] = 0;
  __syncthreads();
  for (int t = threadIdx.x >> 5; t < tokens; t += kSmallThreads / 32) {
    float v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      v[i] = i * 32 + lane < experts ? to_f32<T>(logits[t * pitch + i * 32 + lane])
                                     : -__int_as_float(0x7F800000);
    const Choice c = choose<NV, NV>(v, k, normalize);
    if (lane < k) {
      weights[t * k + lane] = c.weight();
      chosen[t * k + lane] = c.id;
      ids[t * k + lane] = c.id;
      atomicAdd(&base[c.id < 0 ? experts : c.id], 1);
    }
  }
  __syncthreads();
  prefix_counts(base, experts + 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kSmallThreads) offsets[e] = base[e];
  place_slots<kSmallThreads>(
      tokens * k, 0, experts, k, [&](int i) { return ids[i]; }, base, hist, position, rows);
}

// Gradient of the logits: with p the softmax (over the chosen experts
// or over all) and g the gradient of the weights, dl_e = p_e ([e chosen] g_e - sum w g). For
// a chosen expert p_e is its weight. Over all experts the others' p is recomputed from one
// chosen logit: the first chosen one is the largest, m, and its weight is 1 / sum exp(l - m).
// Those p are results of their own, down to e^-87: expf, whose error does not grow with the
// distance (27.6 us, 4.9 TB/s of 134 MB at 65521 x 255 f32; exp_term would take 25.6 and be off
// by up to 62 units of 2^-24). The row is written as if nothing were chosen, then the chosen
// places again.
// LANES lanes a token, at least k; NV experts a lane.
template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(256)
    k_route_backward(const float* __restrict__ dweights, const float* __restrict__ weights,
                     const int32_t* __restrict__ chosen, const T* __restrict__ logits,
                     int64_t tokens, int experts, int64_t pitch, int k, bool normalize,
                     T* __restrict__ dlogits) {
  const int64_t t = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int sub = threadIdx.x % LANES;
  const bool live = t < tokens;
  const T* row = logits + t * pitch;
  T* out = dlogits + t * experts;
  T v[NV];
  if (live && !normalize) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * LANES + sub < experts) v[i] = __ldg(row + i * LANES + sub);
  }
  int id = -1;
  float w = 0.0f, g = 0.0f, m = 0.0f;
  if (live && sub < k) {
    id = chosen[t * k + sub];
    if (id >= 0 && id < experts) {
      w = weights[t * k + sub];
      g = dweights[t * k + sub];
      if (sub == 0 && !normalize) m = to_f32<T>(row[id]);
    } else {
      id = -1;
    }
  }
  float s = w * g;
#pragma unroll
  for (int d = LANES >> 1; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
  m = __shfl_sync(0xFFFFFFFFu, m, 0, LANES);
  // every other weight is 0 where the first is missing, and so is s
  const float scale = -s * __shfl_sync(0xFFFFFFFFu, w, 0, LANES);
  const bool any = __shfl_sync(0xFFFFFFFFu, id, 0, LANES) >= 0;
  if (live) {
    if (normalize || !any) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i * LANES + sub < experts) out[i * LANES + sub] = from_f32<T>(0.0f);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i * LANES + sub < experts)
          out[i * LANES + sub] = from_f32<T>(expf(to_f32<T>(v[i]) - m) * scale);
    }
  }
  __syncwarp();
  if (id >= 0) out[id] = from_f32<T>(w * (g - s));
}

// Registers of logits a lane.
template <typename F>
void with_width(int experts, F&& f) {
  if (experts <= 32) f(std::integral_constant<int, 1>());
  else if (experts <= 64) f(std::integral_constant<int, 2>());
  else if (experts <= 128) f(std::integral_constant<int, 4>());
  else if (experts <= 256) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}

template <typename T>
cudaError_t route_typed(const T* logits, int64_t tokens, int experts, int64_t pitch, int k,
                        bool normalize, float* weights, int32_t* chosen, int32_t* position,
                        int32_t* rows, int32_t* offsets, int32_t* ws, cudaStream_t st) {
  if (tokens <= kSmallTokens) {
    const size_t smem = sizeof(int32_t) * (kSmallTokens * kMaxChosen +
                                           (experts + 1) * (1 + kSmallThreads / 32));
    with_width(experts, [&](auto nv) {
      k_route_small<T, decltype(nv)::value><<<1, kSmallThreads, smem, st>>>(
          logits, (int)tokens, experts, pitch, k, normalize, weights, chosen, position, rows,
          offsets);
    });
    return cudaGetLastError();
  }
  const int block_tokens = select_tokens_of(tokens);
  const int blocks = (int)((tokens + block_tokens - 1) / block_tokens);
  int32_t* totals = ws;
  int32_t* counts = ws + experts + 1;
  with_width(experts, [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    auto deal = [&](auto cn) {
      constexpr int CN = decltype(cn)::value < NV ? decltype(cn)::value : NV;
      k_route_select<T, NV, CN><<<blocks, kSelectThreads, 0, st>>>(
          logits, tokens, experts, pitch, k, normalize, block_tokens, weights, chosen, counts);
    };
    const int most = k * NV;  // candidates of the second stage
    if (most <= 32) deal(std::integral_constant<int, 1>());
    else if (most <= 64) deal(std::integral_constant<int, 2>());
    else if (most <= 128) deal(std::integral_constant<int, 4>());
    else deal(std::integral_constant<int, 8>());
  });
  k_route_scan<<<(experts + 8) / 8, 256, 0, st>>>(counts, totals, experts + 1, blocks);
  const size_t smem = sizeof(int32_t) * (experts + 1) * (1 + kRouteThreads / 32);
  k_route_place<<<blocks, kRouteThreads, smem, st>>>(chosen, counts, totals, tokens, experts, k,
                                                     block_tokens, position, rows, offsets);
  return cudaGetLastError();
}

template <typename F>
cudaError_t with_type(int32_t dtype, F&& f) {
  if (dtype == LGBM_B200_DTYPE_F32) return f(float());
  if (dtype == LGBM_B200_DTYPE_BF16) return f(__nv_bfloat16());
  return f(__half());
}

}  // namespace

int64_t route_workspace(int64_t tokens, int32_t experts, int32_t k) {
  (void)k;
  if (tokens <= kSmallTokens) return 0;
  const int block_tokens = select_tokens_of(tokens);
  const int64_t blocks = (tokens + block_tokens - 1) / block_tokens;
  return (int64_t)sizeof(int32_t) * (experts + 1) * (blocks + 1);
}

cudaError_t launch_route(const void* logits, int32_t dtype, int64_t tokens, int32_t experts,
                         int64_t pitch, int32_t k, bool normalize, float* weights,
                         int32_t* chosen, int32_t* position, int32_t* rows, int32_t* offsets,
                         void* workspace, cudaStream_t st) {
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    return route_typed<T>(static_cast<const T*>(logits), tokens, experts, pitch, k, normalize,
                          weights, chosen, position, rows, offsets,
                          static_cast<int32_t*>(workspace), st);
  });
}

cudaError_t launch_route_backward(const float* dweights, const float* weights,
                                  const int32_t* chosen, const void* logits, int32_t dtype,
                                  int64_t tokens, int32_t experts, int64_t pitch, int32_t k,
                                  bool normalize, void* dlogits, cudaStream_t st) {
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    auto go = [&](auto lanes, auto nv) {
      constexpr int LANES = decltype(lanes)::value;
      const int64_t per_block = 256 / LANES;
      const unsigned blocks = (unsigned)((tokens + per_block - 1) / per_block);
      k_route_backward<T, LANES, decltype(nv)::value><<<blocks, 256, 0, st>>>(
          dweights, weights, chosen, static_cast<const T*>(logits), tokens, experts, pitch, k,
          normalize, static_cast<T*>(dlogits));
      return cudaGetLastError();
    };
    using One = std::integral_constant<int, 1>;
    using Warp = std::integral_constant<int, 32>;
    if (experts <= 4) return go(std::integral_constant<int, 4>(), One());
    if (experts <= 8) return go(std::integral_constant<int, 8>(), One());
    if (experts <= 16) return go(std::integral_constant<int, 16>(), One());
    if (experts <= 32) return go(Warp(), One());
    if (experts <= 64) return go(Warp(), std::integral_constant<int, 2>());
    if (experts <= 128) return go(Warp(), std::integral_constant<int, 4>());
    if (experts <= 256) return go(Warp(), std::integral_constant<int, 8>());
    return go(Warp(), std::integral_constant<int, 16>());
  });
}

}  // namespace experts
}  // namespace lgbm_b200
