// Marks functions that kernels share with the host, in headers that a plain
// C++ compiler takes too.
#pragma once

#ifdef __CUDACC__
#define B2K_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define B2K_HOST_DEVICE inline
#endif
