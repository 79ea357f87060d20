// Gated linear recurrence over time-major (T,B,N), its backward pass and its single step.
//
//   a = sigmoid(f),  h_t = a_t r_t h_{t-1} + c_t z_t,   c = 1 - a (decay_input) or 1,
//   r_t = 0 at a reset, else 1;  a step t >= lengths[b] is the identity and writes 0.
//   backward:  G_t = gh_t + a_{t+1} r_{t+1} G_{t+1},  dz = c G,
//   df = a (1 - a) G (r h_{t-1} - [decay_input] z)  summed over the D = N / G channels of a
//   gate,  dh0 = a_0 r_0 G_0.
//
// Every step is an affine map h -> A h + H of its channel, and maps of consecutive steps
// compose, so time is cut into segments of 16 steps: a warp holds one segment of 32
// channels (one per lane) in registers, the P warps of a block hold P consecutive segments,
// and the blocks of a cluster consecutive runs of those.  Each warp reduces its segment
// to (A, H), the block (then the cluster, over distributed shared memory) folds the maps
// before it in time order, and the warp walks its segment again from the state it found:
// z and f are read once.  The fold's order is fixed, so results do not depend on timing.
// Bound by HBM: 3 elements per channel-step forward, 5 backward.  Backward does not read
// h: the forward keeps the fp32 state before every 16th step (1/16 of an fp32 tensor) and
// each segment recomputes its states from there, which also spares the rounding of a
// 16-bit h.
#pragma once

#include <cooperative_groups.h>

#include "checkpoint8.cuh"
#include "seq_common.cuh"

namespace delrec {

static constexpr int kSeg = 16;        // steps per segment, the distance of the kept states
static constexpr int kScanWarps = 8;   // most segments (warps) per block
static constexpr int kScanCluster = 8; // most blocks per cluster (the portable size)

struct ScanArgs {
  int T, B, N, G, D;
  int decay_input, wide;               // wide: lengths are int64
  int tiles, cpt;                      // channel tiles per row; channels of a tile (<= 32)
  int tph;                             // tiles per gate when D > 32, else 0
  const void *z, *f;
  long long z_t, z_b, f_t, f_b;        // element strides
  const float* h0;
  const void* lengths;
  const uint8_t* resets;               // (T,B)
  void* h;
  long long h_t, h_b;
  float* hT;
  float* states;                       // (ceil(T/16), B, N) or NULL
  int8_t *qz, *qf;                     // 8-bit z (T,B,N) and f (T,B,G) with their exponents
  uint8_t *ez, *ef;
  // backward
  const void* gh;
  long long gh_t, gh_b;
  const float* ghT;
  void *dz, *df;
  long long dz_t, dz_b, df_t, df_b;
  float* dh0;
  float* part;                         // (T,B,G,tph) partial df when D > 32
};

// A channel's place: tile -> (channel, gate).  D = 1: 32 channels; D <= 32: whole gates;
// D > 32: a piece of one gate.
struct Place {
  int c, g;
  bool on;
};
__device__ __forceinline__ Place scan_place(const ScanArgs& p, int tile, int lane) {
  Place r;
  if (p.tph) {
    const int g = tile / p.tph, part = tile - g * p.tph;
    const int d = part * 32 + lane;
    r.g = g;
    r.c = g * p.D + d;
    r.on = d < p.D;
  } else {
    r.c = tile * p.cpt + lane;
    r.on = lane < p.cpt && r.c < p.N;
    r.g = p.D == 1 ? r.c : (r.on ? r.c / p.D : 0);
  }
  return r;
}

// A composed map whose segment holds a reset forgets what came before: A = -0 marks it
// (gates are never negative), so that an infinite or NaN state does not pass through 0 * h.
__device__ __forceinline__ float scan_apply(float2 m, float h) {
  return __float_as_uint(m.x) == 0x80000000u ? m.y : fmaf(m.x, h, m.y);
}

// Folds the (A, H) maps of the block's segments, and of the cluster's blocks, onto the
// running value v: returns the value that enters this warp's segment and moves v on past
// all of them.  rank / warp run in the direction of the recurrence.
template <int P>
struct ScanExchange {
  float2 own[2][P][32];
  float2 all[2][kScanCluster][32];
};
template <int P>
__device__ __forceinline__ float scan_exchange(ScanExchange<P>& sm, int buf, int warp, int lane, int rank, int csize,
                                               float2 m, float& v) {
  namespace cg = cooperative_groups;
  if (P > 1) {
    sm.own[buf][warp][lane] = m;
    __syncthreads();
  }
  if (csize > 1) {
    if (warp == 0) {
      // the block's map, every warp's in turn, into each block of the cluster
      float2 t = m;
      for (int j = 1; j < P; ++j) {
        const float2 n = sm.own[buf][j][lane];
        const bool cut = __float_as_uint(n.x) == 0x80000000u;
        const bool was = __float_as_uint(t.x) == 0x80000000u;
        t = make_float2(cut || was ? -0.f : n.x * t.x, scan_apply(n, t.y));
      }
      cg::cluster_group cl = cg::this_cluster();
      for (int j = 0; j < csize; ++j) {
        ScanExchange<P>* o = cl.map_shared_rank(&sm, j);
        o->all[buf][rank][lane] = t;
      }
    }
    cg::this_cluster().sync();
    float in = v;
    for (int j = 0; j < csize; ++j) {
      if (j == rank) in = v;
      v = scan_apply(sm.all[buf][j][lane], v);
    }
    for (int j = 0; j < warp; ++j) in = scan_apply(sm.own[buf][j][lane], in);
    return in;
  }
  if (P == 1) {
    const float in = v;
    v = scan_apply(m, v);
    return in;
  }
  float in = v;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    if (j == warp) in = v;
    v = scan_apply(sm.own[buf][j][lane], v);
  }
  return in;
}

// One step's coefficients: the gate's product, and the factor of z.
struct StepC {
  float a, om, c;
};
__device__ __forceinline__ StepC scan_coeff(float f, int decay_input) {
  StepC s;
  sigmoid_pair(f, s.a, s.om);
  s.c = decay_input ? s.om : 1.f;
  return s;
}

// PACK (D = 1): also writes z and f in 8 bits; a tile is one group of 32 channels.
template <class T, int P, bool POS, bool PACK>
__global__ void __launch_bounds__(P * 32) k_scan_fwd(ScanArgs p, int csize) {
  __shared__ ScanExchange<P> sm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = csize > 1 ? (int)(blockIdx.x % csize) : 0;
  const int item = blockIdx.x / csize;
  const int b = item / p.tiles, tile = item - b * p.tiles;
  const Place pl = scan_place(p, tile, lane);
  const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
  const T* z = (const T*)p.z + b * p.z_b + pl.c;
  const T* f = (const T*)p.f + b * p.f_b + pl.g;
  T* h = (T*)p.h + b * p.h_b + pl.c;
  float v = (pl.on && p.h0) ? p.h0[(size_t)b * p.N + pl.c] : 0.f;
  const int wave = P * kSeg * csize;
  int buf = 0;
  for (int t0 = 0; t0 < p.T; t0 += wave, buf ^= 1) {
    const int tb = t0 + (rank * P + warp) * kSeg;
    float a[kSeg], x[kSeg];
    float zr[kSeg], fr[kSeg];
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      const int t = tb + i;
      const bool ok = pl.on && t < len;
      zr[i] = ok ? to_f(z[t * p.z_t]) : 0.f;
      fr[i] = ok ? to_f(f[t * p.f_t]) : 0.f;
    }
    float2 m = make_float2(1.f, 0.f);
    bool seen = false;
    unsigned cut = 0;
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      const int t = tb + i;
      const StepC s = scan_coeff(fr[i], p.decay_input);
      a[i] = s.a;
      x[i] = s.c * zr[i];
      if (t >= len) { a[i] = 1.f; x[i] = 0.f; }
      if (PACK && t < p.T) {
        const unsigned ez = q_exponent(__reduce_max_sync(0xffffffffu, q_magnitude(zr[i])));
        const unsigned ef = q_exponent(__reduce_max_sync(0xffffffffu, q_magnitude(fr[i])));
        const size_t row = (size_t)t * p.B + b;
        if (pl.on) {
          p.qz[row * p.N + pl.c] = (int8_t)q_encode(zr[i], q_inverse_scale(ez));
          p.qf[row * p.N + pl.c] = (int8_t)q_encode(fr[i], q_inverse_scale(ef));
        }
        if (lane == 0) {
          p.ez[row * p.tiles + tile] = (uint8_t)ez;
          p.ef[row * p.tiles + tile] = (uint8_t)ef;
        }
      }
      if (POS && p.resets && t < len && p.resets[(size_t)t * p.B + b]) {
        cut |= 1u << i;
        seen = true;
        m = make_float2(0.f, x[i]);
      } else {
        m = make_float2(m.x * a[i], fmaf(a[i], m.y, x[i]));
      }
    }
    if (POS && seen) m.x = -0.f;
    float s = scan_exchange<P>(sm, buf, warp, lane, rank, csize, m, v);
    if (p.states && pl.on && tb < p.T) p.states[((size_t)(tb / kSeg) * p.B + b) * p.N + pl.c] = s;
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      const int t = tb + i;
      s = (POS && ((cut >> i) & 1)) ? x[i] : fmaf(a[i], s, x[i]);
      if (pl.on && t < p.T) h[t * p.h_t] = from_f<T>(t < len ? s : 0.f);
    }
  }
  if (p.hT && pl.on && rank == 0 && warp == 0) p.hT[(size_t)b * p.N + pl.c] = v;
  if (csize > 1) cooperative_groups::this_cluster().sync();   // no block leaves while its peers may still write to it
}

// Sum of v over the lanes of a gate (D <= 32: lanes d = 0 .. D-1 of each gate, the sum in
// lane d = 0; D > 32: the warp's, in lane 0).  A fixed tree.
__device__ __forceinline__ float gate_sum(float v, int d, int D) {
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_down_sync(0xffffffffu, v, o);
    if (d + o < D) v += w;
  }
  return v;
}

// B8: z and f come from their 8-bit form.
template <class T, int P, bool POS, bool B8>
__global__ void __launch_bounds__(P * 32) k_scan_bwd(ScanArgs p, int csize) {
  __shared__ ScanExchange<P> sm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = csize > 1 ? (int)(blockIdx.x % csize) : 0;
  const int item = blockIdx.x / csize;
  const int b = item / p.tiles, tile = item - b * p.tiles;
  const Place pl = scan_place(p, tile, lane);
  const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
  const T* z = (const T*)p.z + b * p.z_b + pl.c;
  const T* f = (const T*)p.f + b * p.f_b + pl.g;
  const T* gh = (const T*)p.gh + b * p.gh_b + pl.c;
  T* dz = (T*)p.dz + b * p.dz_b + pl.c;
  T* df = (T*)p.df + b * p.df_b + pl.g;
  const int gz = (p.N + kQGroup - 1) / kQGroup, gf = (p.G + kQGroup - 1) / kQGroup;
  float v = (pl.on && p.ghT) ? p.ghT[(size_t)b * p.N + pl.c] : 0.f;
  const int wave = P * kSeg * csize;
  const int waves = (p.T + wave - 1) / wave;
  // lane's place inside its gate, for the sums over shared gates
  const int d = p.D == 1 ? 0 : (p.tph ? lane : pl.c - pl.g * p.D);
  const int dn = p.tph ? 32 : p.D;
  int buf = 0;
  for (int wv = waves - 1; wv >= 0; --wv, buf ^= 1) {
    // position in reverse time: block rank 0, warp 0 hold the wave's last segment
    const int pos = (csize - 1 - rank) * P + (P - 1 - warp);
    const int tb = wv * wave + pos * kSeg;
    float zr[kSeg], fr[kSeg], g[kSeg];
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      const int t = tb + i;
      const bool ok = pl.on && t < len;
      if (B8) {
        const size_t row = (size_t)t * p.B + b;
        zr[i] = ok ? q_decode(p.qz[row * p.N + pl.c], q_scale(p.ez[row * gz + pl.c / kQGroup])) : 0.f;
        fr[i] = ok ? (p.qf ? q_decode(p.qf[row * p.G + pl.g], q_scale(p.ef[row * gf + pl.g / kQGroup]))
                           : to_f(f[t * p.f_t]))
                   : 0.f;
      } else {
        zr[i] = ok ? to_f(z[t * p.z_t]) : 0.f;
        fr[i] = ok ? to_f(f[t * p.f_t]) : 0.f;
      }
      g[i] = (ok && p.gh) ? to_f(gh[t * p.gh_t]) : 0.f;
    }
    float s = (pl.on && tb < p.T) ? p.states[((size_t)(tb / kSeg) * p.B + b) * p.N + pl.c] : 0.f;
    unsigned cut = 0;
    float a[kSeg], c[kSeg], e[kSeg];
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      const int t = tb + i;
      const StepC k = scan_coeff(fr[i], p.decay_input);
      if (POS && p.resets && t < len && p.resets[(size_t)t * p.B + b]) {
        cut |= 1u << i;
        s = 0.f;
      }
      a[i] = k.a;
      c[i] = k.c;
      e[i] = k.a * k.om * (p.decay_input ? s - zr[i] : s);
      s = fmaf(k.a, s, k.c * zr[i]);
      if (t >= len) { a[i] = 1.f; c[i] = 0.f; e[i] = 0.f; }
    }
    float2 m = make_float2(1.f, 0.f);
#pragma unroll
    for (int i = kSeg - 1; i >= 0; --i) {
      if (POS && ((cut >> i) & 1)) m = make_float2(0.f, 0.f);
      else m = make_float2(m.x * a[i], a[i] * (m.y + g[i]));
    }
    if (POS && cut) m.x = -0.f;
    float q = scan_exchange<P>(sm, buf, warp, lane, rank, csize, m, v);
#pragma unroll
    for (int i = kSeg - 1; i >= 0; --i) {
      const int t = tb + i;
      const float G = q + g[i];
      q = (POS && ((cut >> i) & 1)) ? 0.f : a[i] * G;
      const bool ok = pl.on && t < p.T;
      if (p.dz && ok) dz[t * p.dz_t] = from_f<T>(t < len ? c[i] * G : 0.f);
      if (p.df) {
        float x = t < len ? e[i] * G : 0.f;
        if (p.D == 1) {
          if (ok) df[t * p.df_t] = from_f<T>(x);
        } else {
          x = gate_sum(pl.on ? x : 0.f, d, dn);
          if (p.tph) {
            if (lane == 0 && t < p.T)
              p.part[(((size_t)t * p.B + b) * p.G + pl.g) * p.tph + (tile - pl.g * p.tph)] = x;
          } else if (ok && d == 0) {
            df[t * p.df_t] = from_f<T>(x);
          }
        }
      }
    }
  }
  if (p.dh0 && pl.on && rank == 0 && warp == 0) p.dh0[(size_t)b * p.N + pl.c] = v;
  if (csize > 1) cooperative_groups::this_cluster().sync();
}

// df[t,b,g] = the sum of its tph partials, in order
template <class T>
__global__ void k_scan_df_sum(ScanArgs p) {
  const size_t n = (size_t)p.T * p.B * p.G;
  for (size_t e = blockIdx.x * (size_t)blockDim.x + threadIdx.x; e < n; e += (size_t)gridDim.x * blockDim.x) {
    const int g = (int)(e % p.G);
    const size_t row = e / p.G;
    const long long b = (long long)(row % p.B), t = (long long)(row / p.B);
    float s = 0.f;
    for (int k = 0; k < p.tph; ++k) s += p.part[e * p.tph + k];
    ((T*)p.df)[t * p.df_t + b * p.df_b + g] = from_f<T>(s);
  }
}

// One time step for every (b, n): h and the next state from z, f and the state (which
// may be updated in place: a thread reads its element before it writes it).
template <class T>
__global__ void __launch_bounds__(128) k_gated_step(int B, int N, int D, int decay_input, const T* __restrict__ z,
                                                    long long z_b, const T* __restrict__ f, long long f_b,
                                                    const float* state, const uint8_t* __restrict__ active,
                                                    T* __restrict__ h, float* next) {
  const size_t n = (size_t)B * N;
  for (size_t e = blockIdx.x * (size_t)blockDim.x + threadIdx.x; e < n; e += (size_t)gridDim.x * blockDim.x) {
    const int b = (int)(e / N), c = (int)(e - (size_t)b * N);
    float s = state ? state[e] : 0.f;
    float o = 0.f;
    if (!active || active[b]) {
      const StepC k = scan_coeff(to_f(f[b * f_b + (D == 1 ? c : c / D)]), decay_input);
      s = fmaf(k.a, s, k.c * to_f(z[b * z_b + c]));
      o = s;
    }
    h[e] = from_f<T>(o);
    next[e] = s;
  }
}

}  // namespace delrec
