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

// x (rows, N) contiguous <-> q (rows, N), e (rows, ceil(N / 32)).  A thread takes V consecutive
// channels of a row (16 bytes of x where rows allow it), so 32 / V lanes hold a group; a
// block covers whole rows of threads side by side (span = lanes of a row, rounded up to whole
// groups), or walks along rows wider than a block, and steps down the rows without divisions, U
// rows in flight.  HBM bounds both: x once, q and e once (64000 x 700 fp32: packed in 47 us,
// restored in 39 to 43, of 35 at the copy rate; registers are held to 40 for 40 warps an SM: more rows in
// flight on fewer warps took longer, and places multiplied out for every row 53).
struct Q8Args {
  long long rows;
  int N, gpr, span, rpb;   // groups and lanes of a row, rows side by side in a block
  const void* x;
  void* out;
  int8_t* q;
  uint8_t* e;
};
template <int V>
__device__ __forceinline__ unsigned group_mask(int lane) {
  constexpr int L = 32 / V;
  return V == 1 ? 0xffffffffu : ((1u << L) - 1u) << (lane & ~(L - 1));
}

template <class T, int V>
__global__ void __launch_bounds__(512, V == 8 ? 2 : 3) k_pack8(Q8Args p) {
  constexpr int L = 32 / V, U = 2;
  const int lane = threadIdx.x & 31;
  const unsigned mask = group_mask<V>(lane);
  const int sub = threadIdx.x / p.span;
  const long long step = (long long)gridDim.x * p.rpb;
  for (int l = threadIdx.x - sub * p.span; l < p.span; l += blockDim.x) {
    const int c = l * V;
    const bool on = c < p.N;
    long long r = blockIdx.x * (long long)p.rpb + sub;
    // places of row r, and from a row to the next one taken
    const T* x = (const T*)p.x + r * p.N + c;
    int8_t* q = p.q + r * p.N + c;
    uint8_t* e = p.e + r * p.gpr + c / kQGroup;
    const long long dn = step * p.N, de = step * p.gpr;
    for (; r < p.rows; r += U * step) {
      VecOf<T, V> raw[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
#pragma unroll
        for (int k = 0; k < V; ++k) raw[j].v[k] = from_f<T>(0.f);
        if (on && r + j * step < p.rows) raw[j] = *(const VecOf<T, V>*)x;
        x += dn;
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (r + j * step < p.rows) {     // the same for the lanes of a group
          float v[V];
          unpack_vec<T, V>(raw[j], v);
          unsigned top = 0;
#pragma unroll
          for (int k = 0; k < V; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
          unsigned ex, code[V];
          if (top < __float_as_uint(kQLargest)) {
            // the sum's low byte is rint(x / s): the quotient is exact, the addition rounds
            ex = q_exponent(top);
            const float inv = q_inverse_scale(ex);
#pragma unroll
            for (int k = 0; k < V; ++k) code[k] = __float_as_uint(fmaf(v[k], inv, 12582912.f));
          } else {
            top = 0;
#pragma unroll
            for (int k = 0; k < V; ++k) top = max(top, q_magnitude(v[k]));
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
            ex = q_exponent(top);
#pragma unroll
            for (int k = 0; k < V; ++k) code[k] = (unsigned)q_encode(v[k], q_inverse_scale(ex));
          }
          if (on) {
            VecOf<int8_t, V> o;
            if constexpr (V % 4 == 0) {
#pragma unroll
              for (int k = 0; k < V; k += 4)
                ((unsigned*)&o)[k / 4] = __byte_perm(__byte_perm(code[k], code[k + 1], 0x0040),
                                                     __byte_perm(code[k + 2], code[k + 3], 0x0040), 0x5410);
            } else {
#pragma unroll
              for (int k = 0; k < V; ++k) o.v[k] = (int8_t)code[k];
            }
            *(VecOf<int8_t, V>*)q = o;
            if (c % kQGroup == 0) *e = (uint8_t)ex;
          }
        }
        q += dn;
        e += de;
      }
    }
  }
}

template <class T, int V>
__global__ void __launch_bounds__(512, V == 8 ? 2 : 3) k_unpack8(Q8Args p) {
  constexpr int U = 2;
  const int sub = threadIdx.x / p.span;
  const long long step = (long long)gridDim.x * p.rpb;
  for (int l = threadIdx.x - sub * p.span; l < p.span; l += blockDim.x) {
    const int c = l * V;
    if (c >= p.N) continue;
    long long r = blockIdx.x * (long long)p.rpb + sub;
    // places of row r, and from a row to the next one taken
    const int8_t* q = p.q + r * p.N + c;
    const uint8_t* e = p.e + r * p.gpr + c / kQGroup;
    T* out = (T*)p.out + r * p.N + c;
    const long long dn = step * p.N, de = step * p.gpr;
    for (; r < p.rows; r += U * step) {
      VecOf<int8_t, V> raw[U];
      uint8_t ex[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (r + j * step < p.rows) {
          raw[j] = *(const VecOf<int8_t, V>*)q;
          ex[j] = *e;
        }
        q += dn;
        e += de;
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (r + j * step < p.rows) {
          const float s = q_scale(ex[j]);
          float v[V];
          bool odd = false;   // a code of an infinity or NaN
#pragma unroll
          for (int k = 0; k < V; ++k) {
            v[k] = (float)raw[j].v[k];
            odd |= fabsf(v[k]) > 126.f;
            v[k] *= s;
          }
          if (odd) {
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = q_decode(raw[j].v[k], s);
          }
          if constexpr (std::is_same_v<T, __half>) {   // saturates, unless the code is an infinity's
#pragma unroll
            for (int k = 0; k < V; ++k)
              if (abs((int)raw[j].v[k]) < 127) v[k] = fminf(fmaxf(v[k], -65504.f), 65504.f);
          }
          *(VecOf<T, V>*)out = pack_vec<T, V>(v);
        }
        out += dn;
      }
    }
  }
}

}  // namespace delrec
