// Shared pieces of the sequence operators (gated scan, block norms, 8-bit checkpoints):
// element types, the sigmoid pair, and the launch macros of their translation unit.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cstdio>
#include <type_traits>

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

// t = exp(-|f|) in [0, 1].  Accurate (2 ulp) for fp32 data; for 16-bit data one product and
// one ex2 (its argument's rounding adds |f| units of 2^-24 to t, far below a 16-bit step).
template <bool ACCURATE>
__device__ __forceinline__ float exp_neg_abs(float f) {
  if (ACCURATE) return expf(-fabsf(f));
  float t;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fabsf(f) * -1.4426950408889634f));
  return t;
}
// The larger and the smaller of sigmoid(f) and sigmoid(-f): 1 / (1 + t) and t / (1 + t),
// each to a few ulp for every f (no cancellation, no overflow).
template <bool ACCURATE>
__device__ __forceinline__ void sigmoid_parts(float f, float& big, float& small) {
  const float t = exp_neg_abs<ACCURATE>(f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(big) : "f"(1.f + t));   // 1 ulp on [1, 2]
  small = t * big;
}
// sg = sigmoid(f), so = 1 - sigmoid(f) = sigmoid(-f)
template <bool ACCURATE>
__device__ __forceinline__ void sigmoid_pair(float f, float& sg, float& so) {
  float big, small;
  sigmoid_parts<ACCURATE>(f, big, small);
  const bool pos = f >= 0.f;
  sg = pos ? big : small;
  so = pos ? small : big;
}
template <class T>
struct Accurate {
  static constexpr bool value = sizeof(T) == 4;
};

// A gate as one register: the smaller of a and 1 - a, signed as f.  The larger is 1 - |w|,
// to one rounding.
template <bool ACCURATE>
__device__ __forceinline__ float gate_fold(float f) {
  float big, small;
  sigmoid_parts<ACCURATE>(f, big, small);
  return f >= 0.f ? small : -small;
}
__device__ __forceinline__ void gate_unfold(float w, float& a, float& om) {
  const float s = fabsf(w), l = 1.f - s;
  const bool pos = !(__float_as_uint(w) >> 31);
  a = pos ? l : s;
  om = pos ? s : l;
}

// V consecutive elements as one aligned access
template <class T, int V>
struct alignas(sizeof(T) * V) VecOf {
  T v[V];
};
// V elements <-> floats; 16-bit ones in pairs (one operation an element to widen, half a one
// to round)
template <class T, int V>
__device__ __forceinline__ void unpack_vec(const VecOf<T, V>& r, float* o) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const unsigned w = ((const unsigned*)&r)[i / 2];
      if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*(const __half2*)&w);
        o[i] = f.x;
        o[i + 1] = f.y;
      } else {
        o[i] = __uint_as_float(w << 16);
        o[i + 1] = __uint_as_float(w & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f(r.v[i]);
  }
}
template <class T, int V>
__device__ __forceinline__ VecOf<T, V> pack_vec(const float* o) {
  VecOf<T, V> r;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (std::is_same_v<T, __half>) ((__half2*)&r)[i / 2] = __floats2half2_rn(o[i], o[i + 1]);
      else ((__nv_bfloat162*)&r)[i / 2] = __floats2bfloat162_rn(o[i], o[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_f<T>(o[i]);
  }
  return r;
}

// lengths (B) int32 or int64; NULL: every row is T long
__device__ __forceinline__ int row_length(const void* lengths, int wide, int b, int T) {
  if (!lengths) return T;
  const long long n = wide ? ((const long long*)lengths)[b] : (long long)((const int*)lengths)[b];
  return n < 0 ? 0 : (n > T ? T : (int)n);
}

static inline int seq_grid(size_t n, int threads, int per_sm) {
  const size_t g = (n + threads - 1) / threads;
  return (int)std::max<size_t>(1, std::min(g, (size_t)kSeqSMs * per_sm));
}

// calls fn(T()) with the element type
template <class F>
static int by_dtype(int dtype, F&& fn) {
  switch (dtype) {
    case DELREC_F32: return fn(float());
    case DELREC_BF16: return fn(__nv_bfloat16());
    case DELREC_F16: return fn(__half());
  }
  return DELREC_ERR_ARG;
}

}  // namespace delrec
