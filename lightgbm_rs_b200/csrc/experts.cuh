// Shared definitions of the expert-layer operators: routing rows to experts, products
// grouped by expert, the combination of the experts' rows, dropout, 4-bit products.
//
// Group offsets, row indices and positions are device data that the host never sees. Every
// kernel therefore clamps the offsets it reads to the rows it was given and skips an index
// outside them: wrong index data give wrong numbers, never an access out of range.
#pragma once

#include <cstdint>
#include <type_traits>

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

// V elements as they lie in memory (V * sizeof(T) is 16, or V is 1), to be loaded first and
// converted later: a conversion right behind its load would wait for it.
template <typename T, int V>
struct Raw {
  uint4 bits;
  __device__ __forceinline__ void load(const T* p) {
    bits = __ldg(reinterpret_cast<const uint4*>(p));
  }
  // The first n of V elements; the others are whatever.
  __device__ __forceinline__ void load_some(const T* p, int n) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 4) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
        else w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + i) << (16 * (i & 1));
      }
    bits = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[V]) {
    uint32_t w[4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 q = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&q);
        } else {
          const __half2 q = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&q);
        }
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct Raw<T, 1> {
  T value;
  __device__ __forceinline__ void load(const T* p) { value = __ldg(p); }
  __device__ __forceinline__ void load_some(const T* p, int) { value = __ldg(p); }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_f32<T>(value); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[1]) {
    *p = from_f32<T>(v[0]);
  }
};

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
  int32_t dtype, grad_dtype;
  const void* x;            // [x_rows, inner]; null where no result needs it
  int64_t x_rows, x_pitch;
  const int32_t* index;     // row of x of every grouped row, or null
  const void* dy;           // [rows, outer], gradients only
  int64_t dy_pitch;
  const void* w;            // [experts, outer, inner]; null where no result needs it
  const int32_t* offsets;
  int64_t rows;
  int32_t experts, inner, outer;
  void *y, *dx, *dw;        // results, null: not wanted
};
int64_t matmul_workspace(const MatmulCall& c);
cudaError_t launch_matmul(const MatmulCall& c, void* workspace, cudaStream_t st);
cudaError_t take_matmul_errors(uint32_t* bits);

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
