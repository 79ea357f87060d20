// Shared pieces of the sequence operators (gated scan, block norms, 8-bit checkpoints):
// element types, the sigmoid pair, and the launch macros of their translation unit.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdio>

#include "../../include/delrec_b200.h"

namespace delrec {

extern unsigned long long g_launches;   // kernels issued by this library (api.cu)

#define SQ_CUDA(call)                                                      \
  do {                                                                     \
    cudaError_t _e = (call);                                               \
    if (_e != cudaSuccess) {                                               \
      fprintf(stderr, "delrec_b200: %s failed: %s\n", #call, cudaGetErrorString(_e)); \
      return DELREC_ERR_CUDA;                                              \
    }                                                                      \
  } while (0)
#define SQ_LAUNCHED()                                                      \
  do {                                                                     \
    ++g_launches;                                                          \
    cudaError_t _e = cudaGetLastError();                                   \
    if (_e != cudaSuccess) {                                               \
      fprintf(stderr, "delrec_b200: launch failed at %s:%d: %s\n", __FILE__, __LINE__, \
              cudaGetErrorString(_e));                                     \
      return DELREC_ERR_CUDA;                                              \
    }                                                                      \
  } while (0)

static constexpr int kSeqSMs = 148;

// element type <-> float (round to nearest even)
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// sg = sigmoid(f), so = 1 - sigmoid(f) = sigmoid(-f), each to a few ulp for every f: from
// t = exp(-|f|) in [0, 1], 1 / (1 + t) and t / (1 + t); no cancellation, no overflow.
__device__ __forceinline__ void sigmoid_pair(float f, float& sg, float& so) {
  const float t = expf(-fabsf(f));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + t));   // 1 ulp on [1, 2]
  const float s = t * r;
  const bool pos = f >= 0.f;
  sg = pos ? r : s;
  so = pos ? s : r;
}

// lengths (B) int32 or int64; NULL: every row is T long
__device__ __forceinline__ int row_length(const void* lengths, int wide, int b, int T) {
  if (!lengths) return T;
  const long long n = wide ? ((const long long*)lengths)[b] : (long long)((const int*)lengths)[b];
  return n < 0 ? 0 : (n > T ? T : (int)n);
}

}  // namespace delrec
