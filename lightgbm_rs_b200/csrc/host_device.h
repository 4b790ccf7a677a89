// Functions of host and device code; a plain C++ compiler takes them as host functions.
#pragma once

#ifdef __CUDACC__
#define LGBM_HOST_DEVICE __host__ __device__ __forceinline__
#define LGBM_UNROLL _Pragma("unroll")
#else
#define LGBM_HOST_DEVICE inline
#define LGBM_UNROLL
#endif
