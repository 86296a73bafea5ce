// Host interface between gn_act.hip (entry points) and gn_one.hip (one pass over the data): false / 0 where the two-launch kernels are to run.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

__attribute__((visibility("hidden"))) size_t gn_one_bytes(int N, long long S, int C, int G);
// would the one-launch form of small images / the one-pass form take 16-byte aligned tensors of this size?
__attribute__((visibility("hidden"))) bool gn_small_takes(int dtype, int N, long long S, int C, int G);
__attribute__((visibility("hidden"))) bool gn_one_takes(int dtype, int N, long long S, int C, int fmt, bool backward);
__attribute__((visibility("hidden"))) bool gn_one_forward(const void* x, int dtype, int vec, int N, long long S, int C, int G, const float* gamma,
                                                          const float* beta, float eps, int act, void* y, float* mean, float* rstd, int fmt,
                                                          uint8_t* codes, uint8_t* scales, void* ws, hipStream_t st);
__attribute__((visibility("hidden"))) bool gn_small_forward(const void* x, int dtype, int vec, int N, long long S, int C, int G, const float* gamma,
                                                            const float* beta, float eps, int act, void* y, float* mean, float* rstd, int fmt,
                                                            uint8_t* codes, uint8_t* scales, hipStream_t st);
__attribute__((visibility("hidden"))) bool gn_one_backward(const void* gy, int dtype, int vec, const void* x, int fmt, const uint8_t* codes,
                                                           const uint8_t* scales, int N, long long S, int C, int G, const float* gamma,
                                                           const float* beta, const float* mean, const float* rstd, int act, void* dx, float* dgamma,
                                                           float* dbeta, void* ws, hipStream_t st);
