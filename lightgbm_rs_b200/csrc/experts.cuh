// Shared definitions of the expert-layer operators: routing rows to experts, products
// grouped by expert, the combination of the experts' rows, dropout, 4-bit products.
//
// Group offsets, row indices and positions are device data that the host never sees. Every
// kernel therefore clamps the offsets it reads to the rows it was given and skips an index
// outside them: wrong index data give wrong numbers, never an access out of range.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "lgbm_b200.h"

namespace lgbm_b200 {

// capi.cu: stores the thread's last error message and returns `code`.
int set_last_error(int code, const char* msg);

namespace experts {

constexpr int kMaxExperts = 512;
constexpr int kMaxChosen = 16;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements as floats; V * sizeof(T) is 16 (one 16-byte access, `p` aligned to
// it) or V is 1.
template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32<T>(*p);
  } else {
    static_assert(V * sizeof(T) == 16, "one 16-byte access");
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32<T>(e[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_f32(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else {
    static_assert(V * sizeof(T) == 16, "one 16-byte access");
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int elem_size(int32_t dtype) { return dtype == LGBM_B200_DTYPE_F32 ? 4 : 2; }

// experts_route.cu
int64_t route_workspace(int64_t tokens, int32_t experts, int32_t k);
cudaError_t launch_route(const void* logits, int32_t dtype, int64_t tokens, int32_t experts,
                         int64_t pitch, int32_t k, bool normalize, float* weights,
                         int32_t* chosen, int32_t* position, int32_t* rows, int32_t* offsets,
                         void* workspace, cudaStream_t st);
cudaError_t launch_route_backward(const float* dweights, const float* weights,
                                  const int32_t* chosen, const void* logits, int32_t dtype,
                                  int64_t tokens, int32_t experts, int64_t pitch, int32_t k,
                                  bool normalize, void* dlogits, cudaStream_t st);

// experts_rows.cu
cudaError_t launch_combine(const void* y, int32_t dtype, int64_t rows, int32_t width,
                           int64_t pitch, const int32_t* position, const float* weights,
                           int64_t tokens, int32_t k, void* out, cudaStream_t st);
cudaError_t launch_combine_backward(const void* dout, const void* y, int32_t dtype,
                                    int64_t rows, int32_t width, int64_t dout_pitch,
                                    int64_t pitch, const int32_t* position,
                                    const float* weights, int64_t tokens, int32_t k, void* dy,
                                    float* dweights, cudaStream_t st);
cudaError_t launch_dropout(const void* x, const void* residual, int32_t dtype, int64_t rows,
                           int64_t width, int64_t pitch, int64_t residual_pitch, uint32_t drop,
                           uint64_t seed, uint64_t offset, void* out, cudaStream_t st);

// experts_matmul.cu
struct MatmulCall {
  int32_t mode;             // 0 forward, 1 input gradient, 2 weight gradient
  int32_t dtype, out_dtype;
  const void* x;            // [x_rows, inner], or null (mode 1)
  int64_t x_rows, x_pitch;
  const int32_t* index;     // row of x of every grouped row, or null
  const void* dy;           // [rows, outer], or null (mode 0)
  int64_t dy_pitch;
  const void* w;            // [experts, outer, inner], or null (mode 2)
  const int32_t* offsets;
  int64_t rows;
  int32_t experts, inner, outer;
  void* out;
};
int64_t matmul_workspace(const MatmulCall& c);
cudaError_t launch_matmul(const MatmulCall& c, void* workspace, cudaStream_t st);
cudaError_t read_matmul_errors(uint32_t* bits);

// experts_few.cu
struct FewCall {
  int32_t dtype;
  const void* x;           // [x_rows, inner]
  int64_t x_rows, x_pitch;
  const int32_t* index;    // row of x of every grouped row, or null
  const void* w;           // [experts, outer, inner], or 4 bits
  int32_t group_size;      // 0: weights of 16 bits, else 32, 64 or 128
  const void* scales;
  const uint8_t* zeros;
  const int32_t* offsets;
  int64_t rows;
  int32_t experts, inner, outer;
  void* y;
};
cudaError_t launch_few(const FewCall& c, cudaStream_t st);

}  // namespace experts
}  // namespace lgbm_b200
