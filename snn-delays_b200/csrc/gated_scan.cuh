// Gated linear recurrence over time-major (T,B,N), its backward pass and its single step.
//
//   a = sigmoid(f),  h_t = a_t r_t h_{t-1} + c_t z_t,   c = 1 - a (decay_input) or 1,
//   r_t = 0 at a reset, else 1;  a step t >= lengths[b] is the identity and writes 0.
//   backward:  G_t = gh_t + a_{t+1} r_{t+1} G_{t+1},  dz = c G,
//   df = a (1 - a) G (r h_{t-1} - [decay_input] z)  summed over the D = N / G channels of a
//   gate,  dh0 = a_0 r_0 G_0.
//
// Every step is an affine map h -> A h + H of its channel, and maps of consecutive steps
// compose, so time is cut into segments: a warp holds one segment (16 steps of 32 V channels,
// V per lane) in registers, the P warps of a block hold P consecutive segments, and the
// blocks of a cluster consecutive runs of those.  Each warp reduces its segment to (A, H),
// the block (then the cluster, over distributed shared memory) folds the maps before it in
// time order, and the warp walks its segment again from the state it found: z and f are
// read once.  The fold's order is fixed, so results do not depend on timing.
//
// Bound by HBM (3 elements per channel-step forward, 5 backward) if the issue slots allow:
// per element there are about 60 (fp32) or 30 (16-bit) of them in the time its bytes
// take, and a straightforward kernel with bounds tests and 64-bit strides spends 80 forward
// and 118 backward.  So 16-bit data goes two channels to a lane with a short exp, strides are
// 32-bit, segments inside a sequence are stored without tests, and the backward's map of
// the reverse recurrence is built in the forward walk (H += g Pi a).  Rows of 16-byte multiples are
// staged: each warp copies its next segment into shared memory (cp.async) while it works on
// the present one, so 16 warps per SM keep the memory busy at 128 registers a thread.  (The plain
// 16-bit backward's 96 KB of stages and 24 of exchange let one block of 8 warps on an SM: it
// is latency-bound.)  Other rows are read an element at a time, which costs half as much again.
// Backward does not read h: the forward keeps the fp32 state before every 16th step (1/16
// of an fp32 tensor) and each segment recomputes its states from there, which also spares
// the rounding of a 16-bit h.  Measured: T=250 B=256 N=512 fp32 forward 72 us (5.6 TB/s, 39
// operations an element), backward 113 us (5.9 TB/s, 65); the same in bf16 41 (5.0 TB/s) and 99 us
// (3.4), fp16 41 and 84; T=784 B=256 N=512 bf16 with 8-bit z and f forward 232 us (47), backward
// 244 us (56, of 44 that its bytes leave time for); one sequence of 65536 steps, N=512 bf16,
// forward 106 us: 16 waves of segments one after another on 16-block clusters.
//
// An infinite state stays infinite or becomes NaN (a product of gates that underflows, times
// infinity) up to the next reset; infinite gradients likewise.
#pragma once

#include <cooperative_groups.h>
#include <string.h>

#include <type_traits>

#include "checkpoint8.cuh"
#include "seq_common.cuh"

namespace delrec {

static constexpr int kSeg = 16;         // steps of a segment, the distance of the kept states
static constexpr int kScanWarps = 8;    // segments (warps) of a block, unless there is one
static constexpr int kScanCluster = 16; // most blocks per cluster (above 8: not every GPU has room)

struct ScanArgs {
  int T, B, N, G, D;
  int decay_input, wide;               // wide: lengths are int64
  int tiles, cpt;                      // channel tiles per row; channels of a tile
  int split;                           // D >= 32: tiles cut across gates, df goes through part
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
  uint8_t* odd;                        // (ceil(T/16), B, groups): infinities or NaN among a segment's codes
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
// channels: 32 V (D = 1, or D >= 32, where it may reach into a second gate), or the whole
// gates that fit 32 lanes (1 < D < 32).
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
    if (warp < csize) {
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
    }
    cl.sync();
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll 4
      for (int j = 0; j < csize; ++j) {
        if (j == rank) in[k] = v[k];
        v[k] = scan_apply<POS>(sm.all[buf][j][k][lane], v[k]);
      }
#pragma unroll
      for (int j = 0; j < P - 1; ++j) {
        const float x = scan_apply<POS>(sm.own[buf][j][k][lane], in[k]);
        if (j < warp) in[k] = x;
      }
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

// A block's shared memory may be written by another block of its cluster only once it has started:
// every block tells so on entry and waits for the others before the first exchange, behind the
// copies of its first segment.
__device__ __forceinline__ void cluster_started(int csize) {
  if (csize > 1) cooperative_groups::this_cluster().barrier_arrive();
}
__device__ __forceinline__ void cluster_wait_started(int csize) {
  if (csize > 1) cooperative_groups::this_cluster().barrier_wait();
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

// ---------------------------------------------------------------------------------
// inputs of a segment
// ---------------------------------------------------------------------------------
// How a kernel gets its inputs.  DIRECT: plain loads, any layout (V = 1).  STAGED: rows copied
// through shared memory ahead of time; a gate per channel, rows and strides of 16-byte
// multiples.  WIDE: D >= 32, plain loads; a tile reaches into two gates at most, so lanes 0-15
// and 16-31 hold the 16 steps of one each and hand them round.
enum : int { SCAN_DIRECT = 0, SCAN_STAGED = 1, SCAN_WIDE = 2 };

template <int BYTES>
struct alignas(BYTES == 16 ? 16 : BYTES) RawBytes {
  char b[BYTES];
};

// S rows of ROWB bytes into shared memory, 16 bytes per copy, stride elements of E apart; rows
// at or past n and columns past the row's end (left bytes) become 0 without being read.
template <int ROWB, int S, class E>
__device__ __forceinline__ void stage_rows(unsigned dst, const E* row0, int stride, int n, int left, int lane) {
  constexpr int CH = ROWB / 16, PER = 32 / CH;   // copies of a row, rows of one round
  const int i0 = lane / CH, c = lane % CH * 16;
  const char* src = (const char*)row0 + c;
  dst += i0 * ROWB + c;
  if (n >= S && left >= ROWB) {
#pragma unroll
    for (int j = 0; j < S; j += PER)
      if (PER <= S || i0 < S)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + j * ROWB),
                     "l"(src + (long long)stride * ((i0 + j) * (int)sizeof(E))));
  } else {
#pragma unroll
    for (int j = 0; j < S; j += PER)
      if (PER <= S || i0 < S) {
        const bool ok = i0 + j < n && c < left;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + j * ROWB),
                     "l"(ok ? src + (long long)stride * ((i0 + j) * (int)sizeof(E)) : (const char*)row0),
                     "r"(ok ? 16 : 0));
      }
  }
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void stage_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// plain loads of a segment's V = 1 channel, 0 at or past n or where the lane is off
template <class E>
__device__ __forceinline__ void direct_rows(const E* base, int stride, int n, bool on, E (&r)[kSeg]) {
  if (on && n >= kSeg) {
#pragma unroll
    for (int i = 0; i < kSeg; ++i) r[i] = *at_step(base, stride, i);
  } else {
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      memset(&r[i], 0, sizeof(E));
      if (on && i < n) r[i] = *at_step(base, stride, i);
    }
  }
}

// A position in a kernel's work: item (row b and channel tile), wave of segments.
struct Cursor {
  int item, b, tile, wv;
  __device__ __forceinline__ void start(int it, int tiles, int first) {
    item = it;
    b = it / tiles;
    tile = it - b * tiles;
    wv = first;
  }
};


// A magnitude as an integer of the same order, 16 bits: a 16-bit float's own bits; of an fp32
// value what its scale depends on, its exponent, one more where its mantissa is past 126 / 64.
__device__ __forceinline__ unsigned q_key(unsigned magnitude_bits) { return (magnitude_bits + 0x3ffffu) >> 23; }
template <class T, int V>
__device__ __forceinline__ unsigned pack_key(const VecOf<T, V>& z, const VecOf<T, V>& f) {
  if constexpr (sizeof(T) == 4) {
    unsigned kz = 0, kf = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      kz = max(kz, __float_as_uint(to_f(z.v[k])) & 0x7fffffffu);
      kf = max(kf, __float_as_uint(to_f(f.v[k])) & 0x7fffffffu);
    }
    return q_key(kz) | q_key(kf) << 16;
  } else if constexpr (V == 2) {
    const unsigned a = *(const unsigned*)&z & 0x7fff7fffu, c = *(const unsigned*)&f & 0x7fff7fffu;
    unsigned r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(__byte_perm(a, c, 0x5410)), "r"(__byte_perm(a, c, 0x7632)));
    return r;
  } else {
    return (*(const unsigned short*)&z & 0x7fffu) | (*(const unsigned short*)&f & 0x7fffu) << 16;
  }
}
// A key's scale key: the biased exponent + 6 (255: not finite, or the scale whose codes are cut).
template <class T>
__device__ __forceinline__ unsigned scale_key(unsigned key) {
  if constexpr (sizeof(T) == 4) return key;
  else if constexpr (std::is_same_v<T, __half>) return q_key(__float_as_uint(__half2float(__ushort_as_half((unsigned short)key))));
  else return q_key(key << 16);
}
__device__ __forceinline__ unsigned q_key_exponent(unsigned key) { return key < 7u ? 1u : key - 6u; }
// Low byte: rint(v / s).  v / s is exact and at most 126, the addition rounds it to even.
__device__ __forceinline__ unsigned q_code(float v, float inv) { return __float_as_uint(fmaf(v, inv, 12582912.f)); }
// both 16-bit halves' maxima
__device__ __forceinline__ unsigned max_u16x2(unsigned a, unsigned b) {
  unsigned r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Maxima (of 16-bit halves) of 16 values over the W = 32 or 16 lanes of a group: a lane returns
// that of value lane % 16.  Each exchange halves the values a lane is concerned with.
template <int W>
__device__ __forceinline__ unsigned group_max16(const unsigned (&x)[16], int lane) {
  unsigned v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool up = lane & 8;
    v[j] = max_u16x2(up ? x[j + 8] : x[j], __shfl_xor_sync(0xffffffffu, up ? x[j] : x[j + 8], 8));
  }
#pragma unroll
  for (int w = 4; w > 0; w >>= 1) {
    const bool up = lane & w;
#pragma unroll
    for (int j = 0; j < w; ++j)
      v[j] = max_u16x2(up ? v[j + w] : v[j], __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + w], w));
  }
  if (W == 32) v[0] = max_u16x2(v[0], __shfl_xor_sync(0xffffffffu, v[0], 16));
  return v[0];
}

// Where a segment's 8-bit form goes.
template <int V>
struct PackOut {
  int8_t *qz, *qf;
  uint8_t *ez, *ef, *odd;
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
// A segment's z and f in 8 bits; n: its steps.  A group is the 32 channels of 32 / V lanes; the
// keys of z and f share a register on their way through the lanes, and lane i of a group
// makes the scales of step i.
template <class T, int V>
__device__ __forceinline__ void scan_pack(const VecOf<T, V> (&zr)[kSeg], const VecOf<T, V> (&fr)[kSeg],
                                          const PackOut<V>& o, int n, bool on, bool group_on, int lane) {
  constexpr int S = kSeg, W = 32 / V;
  const int hl = lane & 15;
  unsigned key[S];
#pragma unroll
  for (int i = 0; i < S; ++i) key[i] = pack_key<T, V>(zr[i], fr[i]);
  const unsigned mine = group_max16<W>(key, lane);
  const unsigned kz = scale_key<T>(mine & 0xffffu), kf = scale_key<T>(mine >> 16);
  const unsigned ez = q_key_exponent(kz), ef = q_key_exponent(kf);
  const float iz = q_inverse_scale(ez), jf = q_inverse_scale(ef);
  const int src = lane & ~(W - 1);
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const float sz = __shfl_sync(0xffffffffu, iz, src + i), sf = __shfl_sync(0xffffffffu, jf, src + i);
    unsigned cz[V], cf[V];
    float zf[V], ff[V];
    unpack_vec<T, V>(zr[i], zf);
    unpack_vec<T, V>(fr[i], ff);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      cz[k] = q_code(zf[k], sz);
      cf[k] = q_code(ff[k], sf);
    }
    if (on && i < n) {
      store_codes<V>(at_step(o.qz, o.stride, i), cz);
      store_codes<V>(at_step(o.qf, o.stride, i), cf);
    }
  }
  const bool teller = group_on && (lane & (W - 1)) < S && hl < n;
  if (teller) {
    o.ez[(long long)hl * o.estride] = (uint8_t)ez;
    o.ef[(long long)hl * o.estride] = (uint8_t)ef;
  }
  const unsigned odd_z = __ballot_sync(0xffffffffu, kz >= 255u), odd_f = __ballot_sync(0xffffffffu, kf >= 255u);
  const bool head = group_on && (lane & (W - 1)) == 0;
  const unsigned group = V == 1 ? 0xffffffffu : 0xffffu << src;
  if (head) *o.odd = ((odd_z | odd_f) & group) != 0;
  if (odd_z) scan_pack_slow<T, V, S>(zr, o.qz, o.ez, o.stride, o.estride, n, on, head);
  if (odd_f) scan_pack_slow<T, V, S>(fr, o.qf, o.ef, o.stride, o.estride, n, on, head);
}

// Sum of v over the lanes of a gate of D < 32 lanes (d: the lane's place in it), in the
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

// ---------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------
// PACK (D = 1): also writes z and f in 8 bits; a tile is V groups of 32 channels.
// R: 16-step pieces of a segment; two (plain staged kernels) where a cluster's exchanges are many.
template <class T, int V, int P, int R, bool POS, bool PACK, int MODE>
struct ScanFwd {
  static constexpr int S = kSeg * R, ROWB = 32 * V * (int)sizeof(T);
  static constexpr int STAGE = MODE == SCAN_STAGED ? 2 * S * ROWB : 0;   // bytes of a warp's segment
  static constexpr int SMEM = 2 * P * STAGE;
  // 16-bit pairs and packing take 128 registers, single channels 80
  static constexpr int WARPS = V == 2 || R == 2 || PACK ? 16 : 24;
};
template <class T, int V, int P, int R, bool POS, bool PACK, bool DI, int MODE>
__global__ void __launch_bounds__(P * 32, ScanFwd<T, V, P, R, POS, PACK, MODE>::WARPS / P) k_scan_fwd(ScanArgs p, int csize) {
  using K = ScanFwd<T, V, P, R, POS, PACK, MODE>;
  constexpr int S = K::S, ROWB = K::ROWB;
  static_assert(R == 1 || (MODE == SCAN_STAGED && !PACK), "longer segments are for plain staged inputs");
  __shared__ ScanExchange<P, V> sm;
  extern __shared__ __align__(16) char stage[];
  cluster_started(csize);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = csize > 1 ? (int)(blockIdx.x % csize) : 0;
  const int seg = rank * P + warp, wave = P * S * csize, waves = (p.T + wave - 1) / wave;
  const int items = p.B * p.tiles, step = gridDim.x / csize;
  char* mine = stage + warp * 2 * K::STAGE;
  // copies the segment of a cursor into half h of this warp's stage
  auto fetch = [&](Cursor c, int h) {
    if (MODE == SCAN_STAGED && c.item < items) {
      const int b = c.b, c0 = c.tile * 32 * V, tb = c.wv * wave + seg * S;
      const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
      const int n = len - tb, left = (p.N - c0) * (int)sizeof(T);
      const unsigned dst = (unsigned)__cvta_generic_to_shared(mine + h * K::STAGE);
      stage_rows<ROWB, S>(dst, (const T*)p.z + b * p.z_b + c0 + (long long)tb * p.z_t, p.z_t, n, left, lane);
      stage_rows<ROWB, S>(dst + S * ROWB, (const T*)p.f + b * p.f_b + c0 + (long long)tb * p.f_t, p.f_t, n, left, lane);
    }
    if (MODE == SCAN_STAGED) stage_commit();
  };
  Cursor cur;
  cur.start((int)blockIdx.x / csize, p.tiles, 0);
  fetch(cur, 0);
  cluster_wait_started(csize);
  float v[V];
  for (int buf = 0; cur.item < items; buf ^= 1) {
    Cursor nxt = cur;
    if (++nxt.wv == waves) nxt.start(cur.item + step, p.tiles, 0);
    __syncwarp();   // all lanes are past their reads of the half that is written now
    fetch(nxt, buf ^ 1);
    const int b = cur.b, tile = cur.tile;
    const Place pl = scan_place<V>(p, tile, lane);
    const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
    const int tb = cur.wv * wave + seg * S, n = len - tb;
    if (cur.wv == 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = (pl.on && p.h0) ? p.h0[(size_t)b * p.N + pl.c + k] : 0.f;
    }
    const unsigned cut = POS ? scan_resets<S>(p, b, tb, len, lane) : 0u;
    if (MODE == SCAN_STAGED) {
      stage_wait<1>();
      __syncwarp();
    }
    float a[S][V], x[S][V];
    float2 m[V];
#pragma unroll
    for (int k = 0; k < V; ++k) m[k] = make_float2(1.f, 0.f);
    if (n > 0) {   // else the identity: past the sequence's end
      VecOf<T, V> zr[S], fr[S];
      float wide = 0.f;
      int edge = 32;
      if constexpr (MODE == SCAN_STAGED) {
        const char* r = mine + buf * K::STAGE + lane * V * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < S; ++i) {
          zr[i] = *(const VecOf<T, V>*)(r + i * ROWB);
          fr[i] = *(const VecOf<T, V>*)(r + (S + i) * ROWB);
        }
      } else {
        static_assert(V == 1 && R == 1, "plain loads take one channel and 16 steps to a lane");
        T r[S];
        direct_rows<T>((const T*)p.z + b * p.z_b + pl.c + (long long)tb * p.z_t, p.z_t, n, pl.on, r);
#pragma unroll
        for (int i = 0; i < S; ++i) zr[i].v[0] = r[i];
        if constexpr (MODE == SCAN_DIRECT) {
          direct_rows<T>((const T*)p.f + b * p.f_b + pl.g + (long long)tb * p.f_t, p.f_t, n, pl.on, r);
#pragma unroll
          for (int i = 0; i < S; ++i) fr[i].v[0] = r[i];
        } else {
          const int g0 = tile * 32 / p.D, g = g0 + (lane >> 4), i = lane & 15;
          edge = (g0 + 1) * p.D - tile * 32;
          const bool ok = g < p.G && i < n;
          wide = gate_fold<Accurate<T>::value>(
              ok ? to_f(((const T*)p.f)[b * p.f_b + g + (long long)(tb + i) * p.f_t]) : 0.f);
        }
      }
      if constexpr (PACK) {
        const size_t row = (size_t)tb * p.B + b;
        const int groups = (p.N + kQGroup - 1) / kQGroup, grp = tile * V + lane * V / 32;
        PackOut<V> o;
        o.qz = p.qz + row * p.N + pl.c; o.qf = p.qf + row * p.N + pl.c;
        o.ez = p.ez + row * groups + grp; o.ef = p.ef + row * groups + grp;
        o.stride = p.B * p.N; o.estride = p.B * groups;
        o.odd = p.odd + ((size_t)(tb / kSeg) * p.B + b) * groups + grp;
        scan_pack<T, V>(zr, fr, o, n, pl.on, grp < groups, lane);
      }
#pragma unroll
      for (int i = 0; i < S; ++i) {
        float w = 0.f;
        if (MODE == SCAN_WIDE) w = __shfl_sync(0xffffffffu, wide, i + (lane >= edge ? 16 : 0));
        float zf[V], ff[V];
        unpack_vec<T, V>(zr[i], zf);
        if (MODE != SCAN_WIDE) unpack_vec<T, V>(fr[i], ff);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float om;
          if (MODE == SCAN_WIDE) gate_unfold(w, a[i][k], om);
          else sigmoid_pair<Accurate<T>::value>(ff[k], a[i][k], om);
          x[i][k] = DI ? om * zf[k] : zf[k];
        }
      }
      if (n < S) {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (i >= n) { a[i][k] = 1.f; x[i][k] = 0.f; }
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
    }
    float s[V];
    scan_exchange<P, V, POS>(sm, buf, warp, lane, rank, csize, m, v, s);
    if (pl.on && tb < p.T) {
      // the state before step i, a multiple of 16
      auto keep = [&](int i) {
        if (p.states && tb + i < p.T) {
          VecOf<float, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) o.v[k] = s[k];
          *(VecOf<float, V>*)(p.states + ((size_t)((tb + i) / kSeg) * p.B + b) * p.N + pl.c) = o;
        }
      };
      T* h = (T*)p.h + b * p.h_b + pl.c + (long long)tb * p.h_t;
      const int nT = p.T - tb;
      if (n >= S) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          if (i % kSeg == 0) keep(i);
#pragma unroll
          for (int k = 0; k < V; ++k)
            s[k] = (POS && ((cut >> i) & 1)) ? x[i][k] : fmaf(a[i][k], s[k], x[i][k]);
          *(VecOf<T, V>*)at_step(h, p.h_t, i) = pack_vec<T, V>(s);
        }
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          if (i % kSeg == 0) keep(i);
          VecOf<T, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            if (i < n) s[k] = (POS && ((cut >> i) & 1)) ? x[i][k] : fmaf(a[i][k], s[k], x[i][k]);
            o.v[k] = from_f<T>(i < n ? s[k] : 0.f);
          }
          if (i < nT) *(VecOf<T, V>*)at_step(h, p.h_t, i) = o;
        }
      }
    }
    if (nxt.wv == 0 && p.hT && pl.on && rank == 0 && warp == 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.hT[(size_t)b * p.N + pl.c + k] = v[k];
    }
    cur = nxt;
  }
  if (MODE == SCAN_STAGED) stage_wait<0>();
  if (csize > 1) cooperative_groups::this_cluster().sync();   // no block leaves while its peers may still write to it
}

// ---------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------
// Code k of a pair as a float without its scale: the byte (offset by 128) as the mantissa of 2^23.
template <int V>
__device__ __forceinline__ float code_value(const RawBytes<V>& r, int k) {
  const unsigned x = V == 2 ? *(const unsigned short*)&r ^ 0x8080u : (unsigned)(uint8_t)r.b[0] ^ 0x80u;
  return __uint_as_float(__byte_perm(x, 0x4b000000u, k ? 0x7651 : 0x7650)) - 8388736.f;
}

// What a backward segment reads: z and f as values or codes, g = gh (staged rows are read from
// shared memory where they are needed, so that they hold no registers), the scales of the
// steps spread over the lanes (lane j: step j, or step j / 2 of group j & 1 for V = 2), this
// lane's share of the gates (WIDE).
template <class T, int V, int S, bool B8, int MODE>
struct ScanIn {
  static constexpr int E = B8 ? 1 : (int)sizeof(T), ROWB = 32 * V * E, ROWG = 32 * V * (int)sizeof(T);
  static constexpr bool STAGED = MODE == SCAN_STAGED;
  using Raw = RawBytes<E * V>;
  const char *zf_row, *g_row;   // this lane's place in the staged rows
  Raw z_[STAGED ? 1 : S], f_[STAGED || MODE == SCAN_WIDE ? 1 : S];
  VecOf<T, V> g_[STAGED ? 1 : S];
  float sz, sf, wide;
  int edge;
  __device__ __forceinline__ Raw z(int i) const {
    if constexpr (STAGED) return *(const Raw*)(zf_row + i * ROWB);
    else return z_[i];
  }
  __device__ __forceinline__ Raw f(int i) const {
    if constexpr (STAGED) return *(const Raw*)(zf_row + (S + i) * ROWB);
    else if constexpr (MODE == SCAN_DIRECT) return f_[i];
    else return f_[0];
  }
  __device__ __forceinline__ VecOf<T, V> g(int i) const {
    if constexpr (STAGED) return *(const VecOf<T, V>*)(g_row + i * ROWG);
    else return g_[i];
  }
};
// The walk of one backward segment in time order: gates w, df factors e, and the segment's map
// of the reverse recurrence, in forward order: G enters at the end times Pi a, and g_i times
// the gates up to i.  PLAIN: all steps are inside the sequence, no code stands for an infinity
// or NaN.
template <class T, int V, int S, bool POS, bool B8, bool DI, int MODE, bool PLAIN>
__device__ __forceinline__ void scan_walk(const ScanArgs& p, const ScanIn<T, V, S, B8, MODE>& r, unsigned cut, int n, int lane,
                                          float (&s)[V], float (&w)[S][V], float (&e)[S][V], float2 (&m)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) m[k] = make_float2(1.f, 0.f);
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float sz = 0.f, sf = 0.f, ww = 0.f;
    if (B8) {
      const int src = V == 1 ? i : 2 * i + (lane >> 4);
      sz = __shfl_sync(0xffffffffu, r.sz, src);
      sf = __shfl_sync(0xffffffffu, r.sf, src);
    }
    if (MODE == SCAN_WIDE) ww = __shfl_sync(0xffffffffu, r.wide, i + (lane >= r.edge ? 16 : 0));
    const auto zi = r.z(i), fi = r.f(i);
    float gf[V], zv[V], fv[V];
    unpack_vec<T, V>(r.g(i), gf);
    if constexpr (!B8) {
      unpack_vec<T, V>(*(const VecOf<T, V>*)&zi, zv);
      if (MODE != SCAN_WIDE) unpack_vec<T, V>(*(const VecOf<T, V>*)&fi, fv);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float zf, ff = 0.f;
      if constexpr (!B8) {
        zf = zv[k];
        if (MODE != SCAN_WIDE) ff = fv[k];
      } else if constexpr (!PLAIN) {
        zf = q_decode((int8_t)zi.b[k], sz);
        ff = q_decode((int8_t)fi.b[k], sf);
      } else {
        zf = code_value<V>(zi, k) * sz;
        ff = code_value<V>(fi, k) * sf;
      }
      float a, om, both;   // both = a (1 - a)
      if (MODE == SCAN_WIDE) {
        gate_unfold(ww, a, om);
        both = a * om;
        w[i][k] = ww;
      } else {
        float big, small;
        sigmoid_parts<Accurate<T>::value>(ff, big, small);
        const bool pos = ff >= 0.f;
        a = pos ? big : small;
        om = pos ? small : big;
        both = big * small;
        w[i][k] = __uint_as_float(__float_as_uint(small) | (__float_as_uint(ff) & 0x80000000u));
      }
      if (POS && ((cut >> i) & 1)) s[k] = 0.f;
      e[i][k] = both * (DI ? s[k] - zf : s[k]);
      s[k] = fmaf(a, s[k], DI ? om * zf : zf);
      if (POS && (cut & ((2u << i) - 1))) {
        m[k].x = 0.f;
      } else if (PLAIN || i < n) {
        m[k].x *= a;
        m[k].y = fmaf(m[k].x, gf[k], m[k].y);
      }
    }
  }
}

// The walk back: q is the gradient that enters the segment's last step.  WHOLE: all its
// steps are inside the sequence.  e[i] becomes df.
template <class T, int V, int S, bool POS, bool DI, bool WHOLE, class In>
__device__ __forceinline__ void scan_walk_back(const ScanArgs& p, const In& r, const float (&w)[S][V],
                                               float (&e)[S][V], float (&q)[V], unsigned cut, int n, int nT, T* dz,
                                               T* df) {
#pragma unroll
  for (int i = S - 1; i >= 0; --i) {
    float gf[V], oz[V], of[V];
    unpack_vec<T, V>(r.g(i), gf);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float a, om;
      gate_unfold(w[i][k], a, om);
      const float G_ = q[k] + gf[k];
      float dzv = DI ? om * G_ : G_, dfv = e[i][k] * G_;
      float nq = (POS && ((cut >> i) & 1)) ? 0.f : a * G_;
      if (!WHOLE && i >= n) { dzv = 0.f; dfv = 0.f; nq = q[k]; }
      q[k] = nq;
      e[i][k] = of[k] = dfv;
      oz[k] = dzv;
    }
    if (WHOLE || i < nT) {
      if (dz) *(VecOf<T, V>*)at_step(dz, p.dz_t, i) = pack_vec<T, V>(oz);
      if (df) *(VecOf<T, V>*)at_step(df, p.df_t, i) = pack_vec<T, V>(of);
    }
  }
}

// B8 (D = 1): z and f come from their 8-bit form.
template <class T, int V, int P, int R, bool B8, int MODE>
struct ScanBwd {
  static constexpr int S = kSeg * R, E = B8 ? 1 : (int)sizeof(T);
  static constexpr int ROWB = 32 * V * E, ROWG = 32 * V * (int)sizeof(T);   // bytes of a row of z or f, of gh
  static constexpr int STAGE = MODE == SCAN_STAGED ? S * (2 * ROWB + ROWG) : 0;
  static constexpr int SMEM = 2 * P * STAGE;
};
template <class T, int V, int P, int R, bool POS, bool B8, bool DI, int MODE>
__global__ void __launch_bounds__(P * 32, 16 / P) k_scan_bwd(ScanArgs p, int csize) {
  using K = ScanBwd<T, V, P, R, B8, MODE>;
  static_assert(R == 1 || (MODE == SCAN_STAGED && !B8), "longer segments are for plain staged inputs");
  using E = std::conditional_t<B8, int8_t, T>;
  constexpr int S = K::S, ROWB = K::ROWB, ROWG = K::ROWG;
  __shared__ ScanExchange<P, V> sm;
  extern __shared__ __align__(16) char stage[];
  cluster_started(csize);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = csize > 1 ? (int)(blockIdx.x % csize) : 0;
  const int wave = P * S * csize, waves = (p.T + wave - 1) / wave;
  // block rank 0, warp 0 hold the wave's last segment: the recurrence runs backward
  const int seg = (csize - 1 - rank) * P + (P - 1 - warp);
  const int items = p.B * p.tiles, step = gridDim.x / csize;
  const int groups = (p.N + kQGroup - 1) / kQGroup;
  char* mine = stage + warp * 2 * K::STAGE;
  // z and f as tensors of E
  const E* zp = B8 ? (const E*)p.qz : (const E*)p.z;
  const E* fp = B8 ? (const E*)p.qf : (const E*)p.f;
  const int z_t = B8 ? p.B * p.N : p.z_t, f_t = B8 ? p.B * p.N : p.f_t;
  const long long z_b = B8 ? p.N : p.z_b, f_b = B8 ? p.N : p.f_b;
  float s_ahead[V], sz_ahead = 0.f, sf_ahead = 0.f;
  int odd_ahead = 0;
  auto scales = [&](int b, int tile, int tb, int n, float& sz, float& sf, int& odd) {
    const int i = lane / V, grp = tile * V + lane % V;
    const bool ok = i < S && i < n && grp < groups;
    const size_t o = ((size_t)(tb + i) * p.B + b) * groups + grp;
    sz = ok ? q_scale(p.ez[o]) : 1.f;
    sf = ok ? q_scale(p.ef[o]) : 1.f;
    const int g0 = tile * V + (lane & (V - 1));
    odd = tb < p.T && g0 < groups ? p.odd[((size_t)(tb / kSeg) * p.B + b) * groups + g0] : 0;
  };
  auto state = [&](int b, const Place& pl, int tb, float (&s)[V]) {
    VecOf<float, V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = 0.f;
    if (pl.on && tb < p.T) o = *(const VecOf<float, V>*)(p.states + ((size_t)(tb / kSeg) * p.B + b) * p.N + pl.c);
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = o.v[k];
  };
  // copies the segment of a cursor into half h of this warp's stage, its state and scales
  // into registers
  auto fetch = [&](Cursor c, int h) {
    if (MODE == SCAN_STAGED && c.item < items) {
      const int b = c.b, tile = c.tile, c0 = tile * 32 * V, tb = c.wv * wave + seg * S;
      const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
      const int n = len - tb, left = p.N - c0;
      const unsigned dst = (unsigned)__cvta_generic_to_shared(mine + h * K::STAGE);
      stage_rows<ROWB, S>(dst, zp + b * z_b + c0 + (long long)tb * z_t, z_t, n, left * K::E, lane);
      stage_rows<ROWB, S>(dst + S * ROWB, fp + b * f_b + c0 + (long long)tb * f_t, f_t, n, left * K::E, lane);
      // without gh its rows become 0; the copies want an aligned address all the same
      const T* gh = p.gh ? (const T*)p.gh + b * p.gh_b + c0 + (long long)tb * p.gh_t : (const T*)zp;
      stage_rows<ROWG, S>(dst + 2 * S * ROWB, gh, p.gh_t, p.gh ? n : 0, left * (int)sizeof(T), lane);
      state(b, scan_place<V>(p, tile, lane), tb, s_ahead);
      if (B8) scales(b, tile, tb, n, sz_ahead, sf_ahead, odd_ahead);
    }
    if (MODE == SCAN_STAGED) stage_commit();
  };
  Cursor cur;
  cur.start((int)blockIdx.x / csize, p.tiles, waves - 1);
  fetch(cur, 0);
  cluster_wait_started(csize);
  float v[V];
  for (int buf = 0; cur.item < items; buf ^= 1) {
    Cursor nxt = cur;
    if (--nxt.wv < 0) nxt.start(cur.item + step, p.tiles, waves - 1);
    const int b = cur.b, tile = cur.tile;
    const Place pl = scan_place<V>(p, tile, lane);
    const int len = POS ? row_length(p.lengths, p.wide, b, p.T) : p.T;
    const int tb = cur.wv * wave + seg * S, n = len - tb, nT = p.T - tb;
    ScanIn<T, V, S, B8, MODE> r;
    r.sz = sz_ahead; r.sf = sf_ahead; r.wide = 0.f; r.edge = 32;
    int odd = odd_ahead;
    float s[V];
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = s_ahead[k];
    __syncwarp();   // all lanes are past their reads of the half that is written now
    fetch(nxt, buf ^ 1);
    if (cur.wv == waves - 1) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = (pl.on && p.ghT) ? p.ghT[(size_t)b * p.N + pl.c + k] : 0.f;
    }
    const unsigned cut = POS ? scan_resets<S>(p, b, tb, len, lane) : 0u;
    r.zf_row = mine + buf * K::STAGE + lane * K::E * V;
    r.g_row = mine + buf * K::STAGE + 2 * S * ROWB + lane * V * (int)sizeof(T);
    if constexpr (MODE == SCAN_STAGED) {
      stage_wait<1>();
      __syncwarp();
    } else {
      static_assert(V == 1, "plain loads take one channel to a lane");
      E x[S];
      T y[S];
      direct_rows<E>(zp + b * z_b + pl.c + (long long)tb * z_t, z_t, n, pl.on, x);
#pragma unroll
      for (int i = 0; i < S; ++i) memcpy(&r.z_[i], &x[i], sizeof(E));
      if constexpr (MODE == SCAN_DIRECT) {
        direct_rows<E>(fp + b * f_b + pl.g + (long long)tb * f_t, f_t, n, pl.on, x);
#pragma unroll
        for (int i = 0; i < S; ++i) memcpy(&r.f_[i], &x[i], sizeof(E));
      }
      direct_rows<T>((const T*)p.gh + b * p.gh_b + pl.c + (long long)tb * p.gh_t, p.gh_t, n, pl.on && p.gh, y);
#pragma unroll
      for (int i = 0; i < S; ++i) r.g_[i].v[0] = y[i];
      state(b, pl, tb, s);
      if (B8) scales(b, tile, tb, n, r.sz, r.sf, odd);
    }
    odd = B8 ? __any_sync(0xffffffffu, odd) : 0;
    if constexpr (MODE == SCAN_WIDE) {
      const int g0 = tile * 32 / p.D, g = g0 + (lane >> 4), i = lane & 15;
      r.edge = (g0 + 1) * p.D - tile * 32;
      const bool ok = g < p.G && i < n;
      r.wide = gate_fold<Accurate<T>::value>(
          ok ? to_f(((const T*)p.f)[b * p.f_b + g + (long long)(tb + i) * p.f_t]) : 0.f);
    }
    float w[S][V], e[S][V];
    float2 m[V];
#pragma unroll
    for (int k = 0; k < V; ++k) m[k] = make_float2(1.f, 0.f);
    if (n > 0) {   // else the identity: past the sequence's end
      if (n >= S && !odd) scan_walk<T, V, S, POS, B8, DI, MODE, true>(p, r, cut, n, lane, s, w, e, m);
      else scan_walk<T, V, S, POS, B8, DI, MODE, false>(p, r, cut, n, lane, s, w, e, m);
    }
    if (POS && cut) {
#pragma unroll
      for (int k = 0; k < V; ++k) m[k].x = -0.f;
    }
    float q[V];
    scan_exchange<P, V, POS>(sm, buf, warp, lane, rank, csize, m, v, q);
    T* dz = pl.on && p.dz ? (T*)p.dz + b * p.dz_b + pl.c + (long long)tb * p.dz_t : nullptr;
    T* df = pl.on && p.df && p.D == 1 ? (T*)p.df + b * p.df_b + pl.c + (long long)tb * p.df_t : nullptr;
    if (n >= S) {
      scan_walk_back<T, V, S, POS, DI, true>(p, r, w, e, q, cut, n, nT, dz, df);
    } else if (n > 0) {
      scan_walk_back<T, V, S, POS, DI, false>(p, r, w, e, q, cut, n, nT, dz, df);
    } else {
      VecOf<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.v[k] = from_f<T>(0.f);
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < nT) {
          if (dz) *(VecOf<T, V>*)at_step(dz, p.dz_t, i) = o;
          if (df) *(VecOf<T, V>*)at_step(df, p.df_t, i) = o;
        }
    }
    if constexpr (MODE == SCAN_WIDE) {
      if (p.df) {
        // the tile's channels of its first gate, and of the one it reaches into
        float x[S];
#pragma unroll
        for (int i = 0; i < S; ++i) x[i] = pl.on && n > 0 && lane < r.edge ? e[i][0] : 0.f;
        const int t = tb + (lane >> 1);
        const float s0 = warp_sum16(x, lane);
        float s1 = 0.f;
        if (r.edge < 32) {
#pragma unroll
          for (int i = 0; i < S; ++i) x[i] = pl.on && n > 0 && lane >= r.edge ? e[i][0] : 0.f;
          s1 = warp_sum16(x, lane);
        }
        if (t < p.T) p.part[(((size_t)t * p.B + b) * p.tiles + tile) * 2 + (lane & 1)] = lane & 1 ? s1 : s0;
      }
    } else if constexpr (MODE == SCAN_DIRECT && !B8) {
      if (p.D > 1 && p.df) {
        T* o = (T*)p.df + b * p.df_b + pl.g + (long long)tb * p.df_t;
        const int d = pl.c - pl.g * p.D;
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const float x = gate_sum(pl.on && n > 0 ? e[i][0] : 0.f, d, p.D);
          if (pl.on && d == 0 && i < nT) *at_step(o, p.df_t, i) = from_f<T>(x);
        }
      }
    }
    if (nxt.wv == waves - 1 && p.dh0 && pl.on && rank == 0 && warp == 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.dh0[(size_t)b * p.N + pl.c + k] = v[k];
    }
    cur = nxt;
  }
  if (MODE == SCAN_STAGED) stage_wait<0>();
  if (csize > 1) cooperative_groups::this_cluster().sync();
}

// df[t,b,g] = the sums of the tiles that gate g spans (D >= 32), in order
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


// ---------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------
struct ScanShape {
  int V, P, R, csize, mode;
  unsigned grid;
};
// the kernels of a direction, by element type (gated_fwd.cu, gated_bwd.cu)
int scan_run_forward(int dtype, ScanArgs& p, const ScanShape& sh, bool pos, cudaStream_t st);
int scan_run_backward(int dtype, ScanArgs& p, const ScanShape& sh, bool pos, cudaStream_t st);

}  // namespace delrec
