// Gated linear recurrence over time-major (T,B,N), its backward pass and its single step.
//
//   a = sigmoid(f),  h_t = a_t r_t h_{t-1} + c_t z_t,   c = 1 - a (decay_input) or 1,
//   r_t = 0 at a reset, else 1;  a step t >= lengths[b] is the identity and writes 0.
//   backward:  G_t = gh_t + a_{t+1} r_{t+1} G_{t+1},  dz = c G,
//   df = a (1 - a) G (r h_{t-1} - [decay_input] z)  summed over the D = N / G channels of a
//   gate,  dh0 = a_0 r_0 G_0.
//
// Every step is an affine map h -> A h + H of its channel, and maps of consecutive steps
// compose, so time is cut into segments: a warp holds one segment (S steps of 32 V channels,
// V per lane) in registers, the P warps of a block hold P consecutive segments, and the
// blocks of a cluster consecutive runs of those.  Each warp reduces its segment to (A, H),
// the block (then the cluster, over distributed shared memory) folds the maps before it in
// time order, and the warp walks its segment again from the state it found: z and f are
// read once.  The fold's order is fixed, so results do not depend on timing.
//
// Bound by HBM (3 elements per channel-step forward, 5 backward) if the issue slots allow:
// per element there are about 60 (fp32) or 30 (16-bit) of them in the time its bytes
// take, and a straightforward kernel with bounds tests and 64-bit strides spends 80 forward
// and 118 backward.  So segments that lie inside a sequence run without tests, strides are 32-bit,
// 16-bit data goes two channels to a lane with a short exp, and the backward's map of the
// reverse recurrence is built in the forward walk (H += g Pi a).  Backward does not read h:
// the forward keeps the fp32 state before every 16th step (1/16 of an fp32 tensor) and each
// segment recomputes its states from there, which also spares the rounding of a 16-bit h.
#pragma once

#include <cooperative_groups.h>

#include "checkpoint8.cuh"
#include "seq_common.cuh"

namespace delrec {

static constexpr int kSeg = 16;         // distance of the kept states; steps of a backward segment
static constexpr int kScanCluster = 16; // most blocks per cluster (above 8: not every GPU has room)

struct ScanArgs {
  int T, B, N, G, D;
  int decay_input, wide;               // wide: lengths are int64
  int tiles, cpt;                      // channel tiles per row; channels of a tile
  int split;                           // D > 32: tiles cut across gates, df goes through part
  int ahead;                           // rows are whole aligned sectors: fetch the next wave to L2
  const void *z, *f;
  int z_t, f_t, h_t;                   // element strides of time
  long long z_b, f_b, h_b;             // and of the batch
  const float* h0;
  const void* lengths;
  const uint8_t* resets;               // (T,B)
  void* h;
  float* hT;
  float* states;                       // (ceil(T/16), B, N) or NULL
  int8_t *qz, *qf;                     // 8-bit z and f (T,B,N) with their exponents
  uint8_t *ez, *ef;
  // backward
  const void* gh;
  int gh_t, dz_t, df_t;
  long long gh_b, dz_b, df_b;
  const float* ghT;
  void *dz, *df;
  float* dh0;
  float* part;                         // (T,B,tiles,2): a tile's df sums of its first and second gate
};

// A lane's place in a tile: its first channel and its gate.  A tile is cpt consecutive
// channels: 32 V (D = 1, or D > 32, where it may reach into a second gate), or the whole
// gates that fit 32 lanes (1 < D <= 32).
struct Place {
  int c, g;
  bool on;
};
template <int V>
__device__ __forceinline__ Place scan_place(const ScanArgs& p, int tile, int lane) {
  Place r;
  r.c = tile * p.cpt + lane * V;
  r.on = lane * V < p.cpt && r.c < p.N;
  if (!r.on) r.c = 0;
  r.g = p.D == 1 ? r.c : r.c / p.D;
  return r;
}

// A composed map whose segment holds a reset forgets what came before: A = -0 marks it
// (gates are never negative), so that an infinite or NaN state does not pass through 0 * h.
template <bool POS>
__device__ __forceinline__ float scan_apply(float2 m, float h) {
  if (POS && __float_as_uint(m.x) == 0x80000000u) return m.y;
  return fmaf(m.x, h, m.y);
}

// Folds the (A, H) maps of the block's segments, and of the cluster's blocks, onto the
// running values v (one per channel of the lane): on return in[] are the values that enter
// this warp's segment and v those past all segments.  rank and warp count in the direction
// of the recurrence.  The buffers alternate, so one barrier per call is enough.
template <int P, int V>
struct ScanExchange {
  float2 own[2][P][V][32];
  float2 all[2][kScanCluster][V][32];
};
template <int P, int V, bool POS>
__device__ __forceinline__ void scan_exchange(ScanExchange<P, V>& sm, int buf, int warp, int lane, int rank, int csize,
                                              const float2 (&m)[V], float (&v)[V], float (&in)[V]) {
  namespace cg = cooperative_groups;
  if (P > 1) {
#pragma unroll
    for (int k = 0; k < V; ++k) sm.own[buf][warp][k][lane] = m[k];
    __syncthreads();
  }
  if (csize > 1) {
    // the block's map, every warp's in turn, into each block of the cluster; the warps
    // share the destinations
    cg::cluster_group cl = cg::this_cluster();
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float2 t = P > 1 ? sm.own[buf][0][k][lane] : m[k];
#pragma unroll
      for (int j = 1; j < P; ++j) {
        const float2 n = sm.own[buf][j][k][lane];
        const bool cut = POS && (__float_as_uint(n.x) == 0x80000000u || __float_as_uint(t.x) == 0x80000000u);
        t = make_float2(cut ? -0.f : n.x * t.x, scan_apply<POS>(n, t.y));
      }
      for (int j = warp; j < csize; j += P) cl.map_shared_rank(&sm, j)->all[buf][rank][k][lane] = t;
    }
    cl.sync();
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float x = v[k], y = v[k];
      for (int j = 0; j < csize; ++j) {
        if (j == rank) x = y;
        y = scan_apply<POS>(sm.all[buf][j][k][lane], y);
      }
      for (int j = 0; j < warp; ++j) x = scan_apply<POS>(sm.own[buf][j][k][lane], x);
      in[k] = x;
      v[k] = y;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    in[k] = v[k];
    if (P == 1) {
      v[k] = scan_apply<POS>(m[k], v[k]);
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        if (j == warp) in[k] = v[k];
        v[k] = scan_apply<POS>(sm.own[buf][j][k][lane], v[k]);
      }
    }
  }
}

// base + i * stride elements: one 32 x 32 -> 64 bit multiply-add (i is a constant)
template <class E>
__device__ __forceinline__ E* at_step(E* base, int stride, int i) {
  return (E*)((char*)base + (long long)stride * (long long)(i * (int)sizeof(E)));
}
template <class E>
__device__ __forceinline__ const E* at_step(const E* base, int stride, int i) {
  return (const E*)((const char*)base + (long long)stride * (long long)(i * (int)sizeof(E)));
}

// bit i: a reset at step tb + i (below n)
template <int S>
__device__ __forceinline__ unsigned scan_resets(const ScanArgs& p, int b, int tb, int n, int lane) {
  if (!p.resets) return 0u;
  const bool r = lane < S && tb + lane < n && p.resets[(size_t)(tb + lane) * p.B + b];
  return __ballot_sync(0xffffffffu, r);
}

// The S x V elements of a segment, 0 past n (bounds) or where the lane is off.
template <class T, int V, int S>
__device__ __forceinline__ void scan_load(const T* base, int stride, int tb, int n, bool on, VecOf<T, V> (&r)[S]) {
  if (on && tb + S <= n) {
#pragma unroll
    for (int i = 0; i < S; ++i) r[i] = *(const VecOf<T, V>*)at_step(base, stride, i);
  } else {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if (on && tb + i < n) {
        r[i] = *(const VecOf<T, V>*)at_step(base, stride, i);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) r[i].v[k] = from_f<T>(0.f);
      }
    }
  }
}

// The biased exponent of a value's 8-bit scale before its offset of 6: the float's own, one
// more where its mantissa is past 126 / 64.  Monotone in |v|, so the group's largest key is
// the key of its largest value.  255: not finite, or at the scale whose codes are cut.
__device__ __forceinline__ unsigned q_key(float v) {
  return ((__float_as_uint(v) & 0x7fffffffu) + 0x3ffffu) >> 23;
}
__device__ __forceinline__ unsigned q_key_exponent(unsigned key) { return key < 7u ? 1u : key - 6u; }
// Low byte: rint(v / s).  v / s is exact and at most 126, the addition rounds it to even.
__device__ __forceinline__ unsigned q_code(float v, unsigned ex) {
  return __float_as_uint(fmaf(v, q_inverse_scale(ex), 12582912.f));
}
// |-| of two 16-bit keys at once
__device__ __forceinline__ unsigned max_u16x2(unsigned a, unsigned b) { return __vmaxu2(a, b); }

// Where a segment's 8-bit form goes.
template <int V>
struct PackOut {
  int8_t *qz, *qf;
  uint8_t *ez, *ef;
  int stride, estride;   // of a time step
};
// V codes of one step and channel pair
template <int V>
__device__ __forceinline__ void store_codes(int8_t* q, const unsigned (&c)[V]) {
  if constexpr (V == 1) *q = (int8_t)c[0];
  else *(uint16_t*)q = (uint16_t)__byte_perm(c[0], c[1], 0x0040);
}
// Segments that hold a value that is not finite, or one at the largest scale: step by step.
template <class T, int V, int S>
__device__ __noinline__ void scan_pack_slow(const VecOf<T, V>* r, int8_t* q, uint8_t* e, int stride, int estride, int n,
                                            bool on, bool head) {
  constexpr int W = 32 / V;
  for (int i = 0; i < S; ++i) {
    unsigned top = 0;
    for (int k = 0; k < V; ++k) top = max(top, q_magnitude(to_f(r[i].v[k])));
    for (int o = W / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const unsigned ex = q_exponent(top);
    unsigned c[V];
    for (int k = 0; k < V; ++k) c[k] = (unsigned)q_encode(to_f(r[i].v[k]), q_inverse_scale(ex));
    if (i < n) {
      if (on) store_codes<V>(at_step(q, stride, i), c);
      if (head) *at_step(e, estride, i) = (uint8_t)ex;
    }
  }
}
// A segment's z and f in 8 bits; n: its steps below T.  A group is the 32 channels of 32 / V
// lanes; the keys of z and f share a register on their way through the lanes.
template <class T, int V, int S>
__device__ __forceinline__ void scan_pack(const VecOf<T, V> (&zr)[S], const VecOf<T, V> (&fr)[S], const PackOut<V>& o,
                                          int n, bool on, bool group_on, int lane) {
  constexpr int W = 32 / V;
  const int hl = lane & (W - 1);
  unsigned mine = 0, top = 0;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float zv[V], fv[V];
    unsigned kz = 0, kf = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      zv[k] = to_f(zr[i].v[k]);
      fv[k] = to_f(fr[i].v[k]);
      kz = max(kz, __float_as_uint(zv[k]) & 0x7fffffffu);
      kf = max(kf, __float_as_uint(fv[k]) & 0x7fffffffu);
    }
    unsigned key = q_key(__uint_as_float(kz)) | q_key(__uint_as_float(kf)) << 16;
#pragma unroll
    for (int s = W / 2; s > 0; s >>= 1) key = max_u16x2(key, __shfl_xor_sync(0xffffffffu, key, s));
    top = max_u16x2(top, key);
    if (hl == i) mine = key;
    const unsigned ez = q_key_exponent(key & 0xffffu), ef = q_key_exponent(key >> 16);
    unsigned cz[V], cf[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      cz[k] = q_code(zv[k], ez);
      cf[k] = q_code(fv[k], ef);
    }
    if (on && i < n) {
      store_codes<V>(at_step(o.qz, o.stride, i), cz);
      store_codes<V>(at_step(o.qf, o.stride, i), cf);
    }
  }
  if (group_on && hl < n && hl < S) {
    o.ez[(long long)hl * o.estride] = (uint8_t)q_key_exponent(mine & 0xffffu);
    o.ef[(long long)hl * o.estride] = (uint8_t)q_key_exponent(mine >> 16);
  }
  const bool head = group_on && hl == 0;
  if (__any_sync(0xffffffffu, (top & 0xffffu) >= 255u))
    scan_pack_slow<T, V, S>(zr, o.qz, o.ez, o.stride, o.estride, n, on, head);
  if (__any_sync(0xffffffffu, (top >> 16) >= 255u))
    scan_pack_slow<T, V, S>(fr, o.qf, o.ef, o.stride, o.estride, n, on, head);
}

// Asks L2 for a segment's rows ahead of their loads: S rows of BYTES, a lane per 32-byte sector.
template <int S, int BYTES, class T>
__device__ __forceinline__ void scan_prefetch(const T* row0, int stride, int n, int lane) {
  constexpr int PER = BYTES / 32;
#pragma unroll
  for (int j = 0; j < S * PER; j += 32) {
    const int i = (j + lane) / PER, s = (j + lane) % PER;
    if (i < n) {
      const char* a = (const char*)(row0 + (long long)i * stride) + s * 32;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a));
    }
  }
}

// PACK (D = 1): also writes z and f in 8 bits; a tile is V groups of 32 channels.
template <class T, int V, int S, int P, bool POS, bool PACK>
__global__ void __launch_bounds__(P * 32, (PACK ? 16 : 24) / P) k_scan_fwd(ScanArgs p, int csize) {
  __shared__ ScanExchange<P, V> sm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = csize > 1 ? (int)(blockIdx.x % csize) : 0;
  const int seg = rank * P + warp, wave = P * S * csize;
  const int items = p.B * p.tiles, step = gridDim.x / csize;
  int buf = 0;
  for (int item = blockIdx.x / csize; item < items; item += step) {
    const int b = item / p.tiles, tile = item - b * p.tiles;
    const Place pl = scan_place<V>(p, tile, lane);
    const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
    const T* z = (const T*)p.z + b * p.z_b + pl.c + (long long)seg * S * p.z_t;
    const T* f = (const T*)p.f + b * p.f_b + pl.g + (long long)seg * S * p.f_t;
    T* h = (T*)p.h + b * p.h_b + pl.c + (long long)seg * S * p.h_t;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = (pl.on && p.h0) ? p.h0[(size_t)b * p.N + pl.c + k] : 0.f;
    for (int t0 = 0; t0 < p.T; t0 += wave, buf ^= 1) {
      const int tb = t0 + seg * S;
      VecOf<T, V> zr[S], fr[S];
      scan_load<T, V, S>(z, p.z_t, tb, len, pl.on, zr);
      scan_load<T, V, S>(f, p.f_t, tb, len, pl.on, fr);
      const unsigned cut = POS ? scan_resets<S>(p, b, tb, len, lane) : 0u;
      if (p.ahead) {
        // the next wave of this item, or the first of the next one
        const bool more = t0 + wave < p.T;
        const int ni = more ? item : item + step;
        if (ni < items) {
          const int nb = ni / p.tiles, nt = ni - nb * p.tiles, tn = (more ? t0 + wave : 0) + seg * S;
          scan_prefetch<S, 32 * V * (int)sizeof(T)>((const T*)p.z + nb * p.z_b + nt * p.cpt + (long long)tn * p.z_t,
                                                    p.z_t, p.T - tn, lane);
          scan_prefetch<S, 32 * V * (int)sizeof(T)>((const T*)p.f + nb * p.f_b + nt * p.cpt + (long long)tn * p.f_t,
                                                    p.f_t, p.T - tn, lane);
        }
      }
      float a[S][V], x[S][V];
      float2 m[V];
#pragma unroll
      for (int k = 0; k < V; ++k) m[k] = make_float2(1.f, 0.f);
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float zf = to_f(zr[i].v[k]);
          float om;
          sigmoid_pair<Accurate<T>::value>(to_f(fr[i].v[k]), a[i][k], om);
          x[i][k] = p.decay_input ? om * zf : zf;
        }
      if (PACK && tb < p.T) {
        const size_t row = (size_t)tb * p.B + b;
        const int groups = (p.N + kQGroup - 1) / kQGroup, grp = tile * V + lane * V / 32;
        PackOut<V> o;
        o.qz = p.qz + row * p.N + pl.c; o.qf = p.qf + row * p.N + pl.c;
        o.ez = p.ez + row * groups + grp; o.ef = p.ef + row * groups + grp;
        o.stride = p.B * p.N; o.estride = p.B * groups;
        scan_pack<T, V, S>(zr, fr, o, p.T - tb, pl.on, grp < groups, lane);
      }
      if (tb + S > len) {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (tb + i >= len) { a[i][k] = 1.f; x[i][k] = 0.f; }
      }
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          if (POS && ((cut >> i) & 1)) m[k] = make_float2(0.f, x[i][k]);
          else m[k] = make_float2(m[k].x * a[i][k], fmaf(a[i][k], m[k].y, x[i][k]));
        }
      if (POS && cut) {
#pragma unroll
        for (int k = 0; k < V; ++k) m[k].x = -0.f;
      }
      float s[V];
      scan_exchange<P, V, POS>(sm, buf, warp, lane, rank, csize, m, v, s);
      if (p.states && pl.on && tb < p.T && tb % kSeg == 0) {
#pragma unroll
        for (int k = 0; k < V; ++k) p.states[((size_t)(tb / kSeg) * p.B + b) * p.N + pl.c + k] = s[k];
      }
      if (pl.on && tb + S <= len) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          VecOf<T, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            s[k] = (POS && ((cut >> i) & 1)) ? x[i][k] : fmaf(a[i][k], s[k], x[i][k]);
            o.v[k] = from_f<T>(s[k]);
          }
          *(VecOf<T, V>*)at_step(h, p.h_t, i) = o;
        }
      } else if (pl.on) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          VecOf<T, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            s[k] = (POS && ((cut >> i) & 1)) ? x[i][k] : fmaf(a[i][k], s[k], x[i][k]);
            o.v[k] = from_f<T>(tb + i < len ? s[k] : 0.f);
          }
          if (tb + i < p.T) *(VecOf<T, V>*)at_step(h, p.h_t, i) = o;
        }
      }
      z += (long long)wave * p.z_t;
      f += (long long)wave * p.f_t;
      h += (long long)wave * p.h_t;
    }
    if (p.hT && pl.on && rank == 0 && warp == 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.hT[(size_t)b * p.N + pl.c + k] = v[k];
    }
  }
  if (csize > 1) cooperative_groups::this_cluster().sync();   // no block leaves while its peers may still write to it
}

// Sum of v over the lanes of a gate of D <= 32 lanes (d: the lane's place in it), in the
// gate's lane 0.  A fixed tree.
__device__ __forceinline__ float gate_sum(float v, int d, int D) {
  for (int o = 16; o > 0; o >>= 1) {
    if (o >= D) continue;
    const float w = __shfl_down_sync(0xffffffffu, v, o);
    if (d + o < D) v += w;
  }
  return v;
}
// Sums of 16 values over the warp's lanes, in a fixed tree: lane 2 i (and 2 i + 1) returns
// the sum of value i.  16 shuffles instead of 80.
__device__ __forceinline__ float warp_sum16(const float (&x)[16], int lane) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool up = lane & 16;
    v[j] = (up ? x[j + 8] : x[j]) + __shfl_xor_sync(0xffffffffu, up ? x[j] : x[j + 8], 16);
  }
#pragma unroll
  for (int w = 4, o = 8; w > 0; w >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < w; ++j)
      v[j] = (up ? v[j + w] : v[j]) + __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + w], o);
  }
  return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

// A gate as one register: the smaller of a and 1 - a, signed as f.  The larger is 1 - |w|,
// to one rounding.
__device__ __forceinline__ void gate_unfold(float w, float& a, float& om) {
  const float s = fabsf(w), l = 1.f - s;
  const bool pos = !(__float_as_uint(w) >> 31);
  a = pos ? l : s;
  om = pos ? s : l;
}

// An 8-bit segment: codes of S x V channels, the scales of its steps spread over the lanes.
template <int V, int S>
struct Scan8 {
  VecOf<int8_t, V> q[S];
  float scale;                         // lane j: of step j (V = 1), of step j / 2, group j & 1 (V = 2)
};
template <int V, int S>
__device__ __forceinline__ void scan_load8(const ScanArgs& p, const int8_t* q, const uint8_t* e, int b, int tb, int n,
                                           int tile, const Place& pl, int lane, Scan8<V, S>& r) {
  const int groups = (p.N + kQGroup - 1) / kQGroup;
  const int step = lane / V, grp = tile * V + lane % V;
  r.scale = 1.f;
  if (step < S && tb + step < n && grp < groups)
    r.scale = q_scale(e[((size_t)(tb + step) * p.B + b) * groups + grp]);
  const int8_t* base = q + ((size_t)tb * p.B + b) * p.N + pl.c;
  const int stride = p.B * p.N;
  if (pl.on && tb + S <= n) {
#pragma unroll
    for (int i = 0; i < S; ++i) r.q[i] = *(const VecOf<int8_t, V>*)at_step(base, stride, i);
  } else {
#pragma unroll
    for (int i = 0; i < S; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) r.q[i].v[k] = 0;
      if (pl.on && tb + i < n) r.q[i] = *(const VecOf<int8_t, V>*)at_step(base, stride, i);
    }
  }
}
// A code as a float without its scale: the byte (offset by 128) as the mantissa of 2^23.
__device__ __forceinline__ float code_value(int8_t q) {
  return __uint_as_float(0x4b000000u | (uint8_t)(q ^ (int8_t)0x80)) - 8388736.f;
}

// The walk of one backward segment in time order: gates w, df factors e, and the segment's map
// of the reverse recurrence, in forward order: G enters at the end times Pi a, and g_i times
// the gates up to i.  SLOW: 8-bit codes may stand for infinities and NaN.
template <class T, int V, bool POS, bool B8, bool SLOW>
__device__ __forceinline__ float scan_walk(const ScanArgs& p, const VecOf<T, V> (&zr)[kSeg], const VecOf<T, V> (&fr)[kSeg],
                                           const VecOf<T, V> (&g)[kSeg], const Scan8<V, kSeg>& z8,
                                           const Scan8<V, kSeg>& f8, unsigned cut, int n, int lane, float (&s)[V],
                                           float (&w)[kSeg][V], float (&e)[kSeg][V], float2 (&m)[V]) {
  float top = 0.f;   // the largest code
#pragma unroll
  for (int k = 0; k < V; ++k) m[k] = make_float2(1.f, 0.f);
#pragma unroll
  for (int i = 0; i < kSeg; ++i) {
    float sz = 0.f, sf = 0.f;
    if (B8) {
      const int src = V == 1 ? i : 2 * i + (lane >> 4);
      sz = __shfl_sync(0xffffffffu, z8.scale, src);
      sf = __shfl_sync(0xffffffffu, f8.scale, src);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float zf, ff;
      if (!B8) {
        zf = to_f(zr[i].v[k]);
        ff = to_f(fr[i].v[k]);
      } else if (SLOW) {
        zf = q_decode(z8.q[i].v[k], sz);
        ff = q_decode(f8.q[i].v[k], sf);
      } else {
        zf = code_value(z8.q[i].v[k]);
        ff = code_value(f8.q[i].v[k]);
        top = fmaxf(top, fmaxf(fabsf(zf), fabsf(ff)));
        zf *= sz;
        ff *= sf;
      }
      float big, small;
      sigmoid_parts<Accurate<T>::value>(ff, big, small);
      const bool pos = ff >= 0.f;
      const float a = pos ? big : small, om = pos ? small : big;
      w[i][k] = pos ? small : -small;
      if (POS && ((cut >> i) & 1)) s[k] = 0.f;
      const float d = p.decay_input ? s[k] - zf : s[k];
      e[i][k] = big * small * d;
      s[k] = fmaf(a, s[k], p.decay_input ? om * zf : zf);
      if (POS && (cut & ((2u << i) - 1))) {
        m[k].x = 0.f;
      } else if (i < n) {
        m[k].x *= a;
        m[k].y = fmaf(m[k].x, to_f(g[i].v[k]), m[k].y);
      }
    }
  }
  return top;
}

// The walk back: q is the gradient that enters the segment's last step.  WHOLE: all its
// steps are inside the sequence.  e[i] becomes df.
template <class T, int V, bool POS, bool WHOLE>
__device__ __forceinline__ void scan_walk_back(const ScanArgs& p, const VecOf<T, V> (&g)[kSeg], const float (&w)[kSeg][V],
                                               float (&e)[kSeg][V], float (&q)[V], unsigned cut, int n, int nT, T* dz,
                                               T* df) {
#pragma unroll
  for (int i = kSeg - 1; i >= 0; --i) {
    VecOf<T, V> oz, of;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float a, om;
      gate_unfold(w[i][k], a, om);
      const float G = q[k] + to_f(g[i].v[k]);
      float dzv = p.decay_input ? om * G : G, dfv = e[i][k] * G;
      float nq = (POS && ((cut >> i) & 1)) ? 0.f : a * G;
      if (!WHOLE && i >= n) { dzv = 0.f; dfv = 0.f; nq = q[k]; }
      q[k] = nq;
      e[i][k] = dfv;
      oz.v[k] = from_f<T>(dzv);
      of.v[k] = from_f<T>(dfv);
    }
    if (WHOLE || i < nT) {
      if (dz) *(VecOf<T, V>*)at_step(dz, p.dz_t, i) = oz;
      if (df) *(VecOf<T, V>*)at_step(df, p.df_t, i) = of;
    }
  }
}

// B8 (D = 1): z and f come from their 8-bit form.
template <class T, int V, int P, bool POS, bool B8>
__global__ void __launch_bounds__(P * 32, 16 / P) k_scan_bwd(ScanArgs p, int csize) {
  constexpr int S = kSeg;
  __shared__ ScanExchange<P, V> sm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = csize > 1 ? (int)(blockIdx.x % csize) : 0;
  const int wave = P * S * csize, waves = (p.T + wave - 1) / wave;
  // block rank 0, warp 0 hold the wave's last segment: the recurrence runs backward
  const int seg = (csize - 1 - rank) * P + (P - 1 - warp);
  const int items = p.B * p.tiles, step = gridDim.x / csize;
  int buf = 0;
  for (int item = blockIdx.x / csize; item < items; item += step) {
    const int b = item / p.tiles, tile = item - b * p.tiles;
    const Place pl = scan_place<V>(p, tile, lane);
    const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
    const long long first = (long long)(waves - 1) * wave + (long long)seg * S;
    const T* z = (const T*)p.z + b * p.z_b + pl.c + first * p.z_t;
    const T* f = (const T*)p.f + b * p.f_b + pl.g + first * p.f_t;
    const T* gh = (const T*)p.gh + b * p.gh_b + pl.c + first * p.gh_t;
    T* dz = (T*)p.dz + b * p.dz_b + pl.c + first * p.dz_t;
    T* df = (T*)p.df + b * p.df_b + pl.g + first * p.df_t;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = (pl.on && p.ghT) ? p.ghT[(size_t)b * p.N + pl.c + k] : 0.f;
    for (int wv = waves - 1; wv >= 0; --wv, buf ^= 1) {
      const int tb = wv * wave + seg * S;
      VecOf<T, V> zr[S], fr[S], g[S];
      Scan8<V, S> z8, f8;
      if (B8) {
        scan_load8<V, S>(p, p.qz, p.ez, b, tb, len, tile, pl, lane, z8);
        scan_load8<V, S>(p, p.qf, p.ef, b, tb, len, tile, pl, lane, f8);
      } else {
        scan_load<T, V, S>(z, p.z_t, tb, len, pl.on, zr);
        scan_load<T, V, S>(f, p.f_t, tb, len, pl.on, fr);
      }
      scan_load<T, V, S>(gh, p.gh_t, tb, len, pl.on && p.gh, g);
      float s[V];
#pragma unroll
      for (int k = 0; k < V; ++k)
        s[k] = (pl.on && tb < p.T) ? p.states[((size_t)(tb / kSeg) * p.B + b) * p.N + pl.c + k] : 0.f;
      const unsigned cut = POS ? scan_resets<S>(p, b, tb, len, lane) : 0u;
      if (p.ahead) {
        // the next wave of this item, or the first of the next one
        const int ni = wv > 0 ? item : item + step;
        if (ni < items) {
          const int nb = ni / p.tiles, nt = ni - nb * p.tiles, tn = (wv > 0 ? wv - 1 : waves - 1) * wave + seg * S;
          constexpr int R = 32 * V * (int)sizeof(T);
          if (B8) {
            const long long o = ((long long)tn * p.B + nb) * p.N + nt * p.cpt;
            scan_prefetch<S, 32 * V>(p.qz + o, p.B * p.N, p.T - tn, lane);
            scan_prefetch<S, 32 * V>(p.qf + o, p.B * p.N, p.T - tn, lane);
          } else {
            scan_prefetch<S, R>((const T*)p.z + nb * p.z_b + nt * p.cpt + (long long)tn * p.z_t, p.z_t, p.T - tn, lane);
            scan_prefetch<S, R>((const T*)p.f + nb * p.f_b + nt * p.cpt + (long long)tn * p.f_t, p.f_t, p.T - tn, lane);
          }
          if (p.gh)
            scan_prefetch<S, R>((const T*)p.gh + nb * p.gh_b + nt * p.cpt + (long long)tn * p.gh_t, p.gh_t, p.T - tn,
                                lane);
        }
      }
      float w[S][V], e[S][V];
      float2 m[V];
      const int n = len - tb, nT = p.T - tb;
      const float top = n >= S ? scan_walk<T, V, POS, B8, false>(p, zr, fr, g, z8, f8, cut, S, lane, s, w, e, m)
                               : scan_walk<T, V, POS, B8, false>(p, zr, fr, g, z8, f8, cut, n, lane, s, w, e, m);
      if (B8 && __any_sync(0xffffffffu, top > 126.f)) {
        // rare: infinities or NaN among the codes; all is read again, so that nothing is kept for it
        scan_load8<V, S>(p, p.qz, p.ez, b, tb, len, tile, pl, lane, z8);
        scan_load8<V, S>(p, p.qf, p.ef, b, tb, len, tile, pl, lane, f8);
#pragma unroll
        for (int k = 0; k < V; ++k)
          s[k] = (pl.on && tb < p.T) ? p.states[((size_t)(tb / kSeg) * p.B + b) * p.N + pl.c + k] : 0.f;
        scan_walk<T, V, POS, B8, true>(p, zr, fr, g, z8, f8, cut, n, lane, s, w, e, m);
      }
      if (POS && cut) {
#pragma unroll
        for (int k = 0; k < V; ++k) m[k].x = -0.f;
      }
      float q[V];
      scan_exchange<P, V, POS>(sm, buf, warp, lane, rank, csize, m, v, q);
      T* dzp = pl.on ? (T*)p.dz : nullptr;
      T* dfp = pl.on && p.D == 1 ? (T*)p.df : nullptr;
      if (dzp) dzp = dz;
      if (dfp) dfp = df;
      if (n >= S) scan_walk_back<T, V, POS, true>(p, g, w, e, q, cut, n, nT, dzp, dfp);
      else scan_walk_back<T, V, POS, false>(p, g, w, e, q, cut, n, nT, dzp, dfp);
      if (V == 1 && p.D > 1 && p.df) {
        if (p.split) {
          // the tile's channels of its first gate, and of the one it reaches into
          const int g0 = tile * 32 / p.D, edge = (g0 + 1) * p.D - tile * 32;
          float x[S];
#pragma unroll
          for (int i = 0; i < S; ++i) x[i] = pl.on && lane < edge ? e[i][0] : 0.f;
          const int t = tb + (lane >> 1);
          const float s0 = warp_sum16(x, lane);
          float s1 = 0.f;
          if (edge < 32) {
#pragma unroll
            for (int i = 0; i < S; ++i) x[i] = pl.on && lane >= edge ? e[i][0] : 0.f;
            s1 = warp_sum16(x, lane);
          }
          if (t < p.T) p.part[(((size_t)t * p.B + b) * p.tiles + tile) * 2 + (lane & 1)] = lane & 1 ? s1 : s0;
        } else {
          const int d = pl.c - pl.g * p.D;
#pragma unroll
          for (int i = 0; i < S; ++i) {
            const float x = gate_sum(pl.on ? e[i][0] : 0.f, d, p.D);
            if (pl.on && d == 0 && tb + i < p.T) *at_step(df, p.df_t, i) = from_f<T>(x);
          }
        }
      }
      z -= (long long)wave * p.z_t;
      f -= (long long)wave * p.f_t;
      gh -= (long long)wave * p.gh_t;
      dz -= (long long)wave * p.dz_t;
      df -= (long long)wave * p.df_t;
    }
    if (p.dh0 && pl.on && rank == 0 && warp == 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.dh0[(size_t)b * p.N + pl.c + k] = v[k];
    }
  }
  if (csize > 1) cooperative_groups::this_cluster().sync();
}

// df[t,b,g] = the sums of the tiles that gate g spans (D > 32), in order
template <class T>
__global__ void k_scan_df_sum(ScanArgs p) {
  const size_t n = (size_t)p.T * p.B * p.G;
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
    const int g = (int)(i % p.G);
    const size_t row = i / p.G;
    const long long b = (long long)(row % p.B), t = (long long)(row / p.B);
    const int lo = g * p.D / 32, hi = ((g + 1) * p.D - 1) / 32;
    float s = 0.f;
    for (int k = lo; k <= hi; ++k) s += p.part[(row * p.tiles + k) * 2 + (k * 32 / p.D == g ? 0 : 1)];
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
      float a, om;
      sigmoid_pair<Accurate<T>::value>(to_f(f[b * f_b + (D == 1 ? c : c / D)]), a, om);
      const float x = to_f(z[b * z_b + c]);
      s = fmaf(a, s, decay_input ? om * x : x);
      o = s;
    }
    h[e] = from_f<T>(o);
    next[e] = s;
  }
}

}  // namespace delrec
