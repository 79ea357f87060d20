// 8-bit checkpoints: rows of N channels in groups of 32 consecutive channels (the last
// group of a row may be shorter), each group with one power-of-two scale 2^(e - 127).
//
//   s = the smallest power of two >= 2^-126 with max |x| <= 126 s  (over the finite x)
//   q = rint(x / s), ties to even: |q| <= 126;   q = 127: +inf, -127: -inf, -128: NaN
//   (at s = 2^122, the largest, |q| <= 63: 64 s is past the largest float)
//
// A power of two makes x / s exact, so q does not depend on how the quotient is
// evaluated; it costs half a bit of the eight on average against max / 127.  A restored
// value has 7 significant bits, so bf16 carries it exactly.  0 / 1 spike trains come back
// exactly (s = 1/64, q = 64).
#pragma once

#include <math_constants.h>

#include "seq_common.cuh"

namespace delrec {

static constexpr int kQGroup = 32;
static constexpr float kQLargest = 63.f * 0x1p122f;

// biased scale exponent (1 .. 249) from the bits of the group's largest finite magnitude
__device__ __forceinline__ unsigned q_exponent(unsigned amax_bits) {
  // 2^k <= amax < 2^(k+1): amax / 2^(k-6) in [64, 128); above 126 (mantissa > 1.96875) one up
  const int k = (int)(amax_bits >> 23) - 6 + ((amax_bits & 0x7fffffu) > 0x7c0000u ? 1 : 0);
  return k < 1 ? 1u : (unsigned)k;
}
__device__ __forceinline__ float q_inverse_scale(unsigned e) { return __uint_as_float((254u - e) << 23); }
__device__ __forceinline__ float q_scale(unsigned e) { return __uint_as_float(e << 23); }
// bits of |x|, 0 for infinities and NaN (what the group's maximum is taken over)
__device__ __forceinline__ unsigned q_magnitude(float x) {
  const unsigned u = __float_as_uint(x) & 0x7fffffffu;
  return u >= 0x7f800000u ? 0u : u;
}
__device__ __forceinline__ int q_encode(float x, float inv) {
  const unsigned u = __float_as_uint(x) & 0x7fffffffu;
  if (u >= 0x7f800000u) return u > 0x7f800000u ? -128 : (x > 0.f ? 127 : -127);
  // |x| >= 63.5 * 2^122 (the scale is then 2^122) stays at 63 steps
  return __float2int_rn(fminf(fmaxf(x, -kQLargest), kQLargest) * inv);
}
__device__ __forceinline__ float q_decode(int q, float s) {
  if (q >= 127 || q <= -127)
    return q == 127 ? CUDART_INF_F : (q == -127 ? -CUDART_INF_F : CUDART_NAN_F);
  return (float)q * s;
}

// A restored value in type T; fp16 saturates at its largest value.
template <class T>
__device__ __forceinline__ T q_store(float v, int q) {
  return from_f<T>(v);
}
template <>
__device__ __forceinline__ __half q_store<__half>(float v, int q) {
  return __float2half_rn(q >= 127 || q <= -127 ? v : fminf(fmaxf(v, -65504.f), 65504.f));
}

// x (rows, N) contiguous -> q (rows, N), e (rows, ceil(N / 32)): a warp per group, a lane
// per channel.
template <class T>
__global__ void __launch_bounds__(256) k_pack8(long long groups, int gpr, int N, const T* __restrict__ x,
                                               int8_t* __restrict__ q, uint8_t* __restrict__ e) {
  const int lane = threadIdx.x & 31;
  const long long stride = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long g = blockIdx.x * (long long)(blockDim.x >> 5) + (threadIdx.x >> 5); g < groups; g += stride) {
    const long long row = g / gpr;
    const int c = (int)(g - row * gpr) * kQGroup + lane;
    const bool on = c < N;
    const float v = on ? to_f(x[row * N + c]) : 0.f;
    const unsigned ex = q_exponent(__reduce_max_sync(0xffffffffu, q_magnitude(v)));
    if (on) q[row * N + c] = (int8_t)q_encode(v, q_inverse_scale(ex));
    if (lane == 0) e[g] = (uint8_t)ex;
  }
}

template <class T>
__global__ void __launch_bounds__(256) k_unpack8(long long groups, int gpr, int N, const int8_t* __restrict__ q,
                                                 const uint8_t* __restrict__ e, T* __restrict__ x) {
  const int lane = threadIdx.x & 31;
  const long long stride = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long g = blockIdx.x * (long long)(blockDim.x >> 5) + (threadIdx.x >> 5); g < groups; g += stride) {
    const long long row = g / gpr;
    const int c = (int)(g - row * gpr) * kQGroup + lane;
    if (c < N) {
      const int v = q[row * N + c];
      x[row * N + c] = q_store<T>(q_decode(v, q_scale(e[g])), v);
    }
  }
}

}  // namespace delrec
