// Selective state space scan and its gradients.  Per channel n of group g and state s:
//
//   delta_t = softplus(dt_t + dt_bias)                      (or dt_t + dt_bias)
//   h_t[s]  = exp(delta_t A[s]) h_{t-1}[s] + delta_t B_t[s] x_t
//   y_t     = (sum_s C_t[s] h_t[s] + D x_t) silu(gate_t)
//
// A thread holds 2 channels x 4 states; L lanes (4 L >= S) share a channel's states, the other
// 32 / L lane groups of a warp hold other channels.  The sums over states (y, dx, ddt) run over four
// values in the thread and then over L lanes, those over channels (dB, dC) over two values and then
// over 32 / L lanes: either way a lane hands on half of what it holds at each exchange.  A block walks
// kSelSeg steps at a time, whose inputs it lays out in shared memory in float32; states stay in registers.
//
// The backward pass keeps the states before every kSelSeg-th step (written by the forward pass),
// recomputes those in between into shared memory and walks the segment back.  Where the rows are
// few, time is cut into chunks: their affine maps come first (LOCAL passes; the product of a chunk's
// decays is exp(A sum delta)), are joined in time order (k_sel_join), and then every chunk runs from
// its own start.
//
// exp(delta A) is ex2((delta log2 e) A): the factor goes with delta, whose rounding differs from step to
// step, not with A, whose rounding would pull every step of a state the same way (the state after 500
// bf16 steps on average 7.9e-7 -> 3.6e-7 off).
//
// What bounds it.  At T=250 B=256 N=512 S=16 fp32 the forward kernel takes 300 us (its bytes, the kept
// states among them, 120; the exponentials, 16 a clock and SM, 116), the backward kernel 850 (180 and 233).
// Both are held up by shared memory and by waiting: 21 and 67 wavefronts a warp, step and 256 states (a
// 16-byte read by 32 lanes is four, however many of them read the same), 73 and 250 instructions, on 20 and
// 12 warps an SM, as many as their registers allow.  Of four channels by four states to a thread (fewer
// reads of B and C, 255 registers: 886 to 1090), the states or the decays of half a segment in registers
// (862 to 1240) and keeping every other state (846 to 909) none was faster backward.  Sums and states are
// float32.
//
// A lane holds four states whether they are there or not, and a power of two of lanes a channel: the time goes in
// steps at S = 4, 8, 16, .. (that fp32 case, forward and backward: S = 1 to 4 215 and 740 us, 5 to 8 230 and 655, 9 to 16
// 270 and 830, 17 to 32 550 and 1750, 33 to 64 1130 and 4560).  S <= 4 is slower backward than 8: k_sel_bwd<float, 1>
// has 255 registers and spills 172 bytes.
#pragma once

#include "f32x2.cuh"
#include "seq_common.cuh"

namespace delrec {

constexpr int kSelSeg = 8;       // steps of a segment; distance of the states kept for the backward pass
constexpr int kSelMaxS = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct SelArgs {
  int T, B, N, S, G, Dg;          // Dg = N / G channels to a group
  int softplus, wide, vec, bcvec; // vec: rows of x, dt, gate, y and their gradients in fours, twos or ones; bcvec: B and C in fours
  int chunks, steps, tiles;       // chunks of `steps` rows; tiles of channels to a group in this launch
  int parts;                      // tiles of a backward launch
  int tile0, add;                 // the first tile; add: dB and dC hold the sums of the launches before
  const void *x, *dt, *Bm, *Cm, *gate;
  const float *A, *D, *bias, *h0;
  const void* lengths;
  const uint8_t* resets;
  void* y;
  float *hT, *states;             // states (ceil(T / kSelSeg), B, N, S)
  long long x_t, x_b, dt_t, dt_b, u_t, u_b, y_t, y_b, bm_t, bm_b, cm_t, cm_b;
  // maps of the chunks: loc (chunks,B,N,S), sumd (chunks,B,N), cut (chunks,B)
  float *loc, *sumd;
  uint8_t* cut;
  // backward
  const void* gy;
  const float* ghT;
  void *dx, *ddt, *dgate;
  float *dh0, *dA, *dD, *db;      // dA (chunks * B, N, S), dD, db (chunks * B, N): partial sums
  float *dB, *dC;                 // (tiles of a launch, T, B, G, S): partial sums
  long long gy_t, gy_b, dx_t, dx_b, ddt_t, ddt_b, du_t, du_b;
};

__device__ __forceinline__ float sel_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ f2 exp22(f2 v) {
  float a, b;
  split(v, a, b);
  return pair(sel_exp2(a), sel_exp2(b));
}
// exp(delta A) from d = delta log2(e).  ex2.approx is low by 2.1e-8 of its value on average (it cuts
// off), and a state that lives for a thousand steps sees that a thousand times: the exponent takes
// 2.1e-8 log2(e) more (a product and a sum cost what a product costs).  d = 0 still gives exactly 1.
constexpr float kSelLow = 2.97e-8f;
__device__ __forceinline__ f2 sel_decay2(f2 d, f2 A) { return exp22(fma2(d, A, pair(kSelLow, kSelLow))); }
// A as the kernels take it: -inf is the lowest number there is, whose decay over any step is the same 0, so that
// delta = 0 (rows past the end, chunks without steps) leaves a state as it is: 0 A is not NaN.  (A NaN stays one.)
__device__ __forceinline__ float sel_finite(float A) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(A), "f"(-3.402823466e38f));
  return r;
}
__device__ __forceinline__ float sel_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// delta and its derivative by dt.  softplus(z) = max(z, 0) + log1p(t), t = exp(-|z|), with log1p(t) =
// 2 artanh(s), s = t / (2 + t) <= 1/3, by its series up to s^15 (what is left out is below 2^-28 of it).
template <class T, bool GRAD>
__device__ __forceinline__ float sel_delta(float z, int softplus, float& d) {
  if (!softplus) {
    d = 1.f;
    return z;
  }
  const float t = exp_neg_abs<Accurate<T>::value>(z), s = t * sel_rcp(2.f + t), q = s * s;
  if (GRAD) {
    const float r = sel_rcp(1.f + t);
    d = z >= 0.f ? r : t * r;
  }
  float p = fmaf(q, 1.f / 15, 1.f / 13);
  p = fmaf(q, p, 1.f / 11);
  p = fmaf(q, p, 1.f / 9);
  p = fmaf(q, p, 1.f / 7);
  p = fmaf(q, p, 1.f / 5);
  p = fmaf(q, p, 1.f / 3);
  const float s2 = s + s;
  return fmaxf(z, 0.f) + fmaf(s2 * q, p, s2);
}

// W elements of the element type as they lie in memory, in whole registers: a load on its way is not
// touched before it is needed
template <class T, int W>
struct RawOf {
  uint32_t w[W * sizeof(T) / 4];
};
// how: 2 all W at once, 1 in pairs (an even number of them is there), 0 one by one
template <class T, int W>
__device__ __forceinline__ void sel_load(RawOf<T, W>& r, const T* p, int how, int left) {
  if (how == 2) {
    constexpr int B = W * sizeof(T);
    if constexpr (B == 16) {
      const uint4 v = *(const uint4*)p;
      r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else if constexpr (B == 8) {
      const uint2 v = *(const uint2*)p;
      r.w[0] = v.x; r.w[1] = v.y;
    } else {
      r.w[0] = *(const uint32_t*)p;
    }
  } else if (how == 1) {
#pragma unroll
    for (int i = 0; i < W; i += 2) {
      if constexpr (sizeof(T) == 4) {
        const uint2 v = i < left ? *(const uint2*)(p + i) : make_uint2(0u, 0u);
        r.w[i] = v.x; r.w[i + 1] = v.y;
      } else {
        r.w[i / 2] = i < left ? *(const uint32_t*)(p + i) : 0u;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 4) {
        r.w[i] = i < left ? ((const uint32_t*)p)[i] : 0u;
      } else {
        const uint32_t v = i < left ? ((const unsigned short*)p)[i] : 0u;
        r.w[i / 2] = i & 1 ? r.w[i / 2] | v << 16 : v;
      }
    }
  }
}
template <class T, int W>
__device__ __forceinline__ void sel_floats(const RawOf<T, W>& r, float* v) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(r.w[i]);
    else if constexpr (std::is_same_v<T, __half>) v[i] = __half2float(__ushort_as_half((unsigned short)(r.w[i / 2] >> 16 * (i & 1))));
    else v[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
  }
}
template <class T, int W>
__device__ __forceinline__ void sel_store(T* p, int how, int left, const float* v) {
  if (how == 2) {
    *(VecOf<T, W>*)p = pack_vec<T, W>(v);
  } else if (how == 1) {
#pragma unroll
    for (int i = 0; i < W; i += 2)
      if (i < left) *(VecOf<T, 2>*)(p + i) = pack_vec<T, 2>(v + i);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) p[i] = from_f<T>(v[i]);
  }
}
__device__ __forceinline__ float4 f4(const float* v) { return make_float4(v[0], v[1], v[2], v[3]); }
// v[i] <- v[i ^ x]
__device__ __forceinline__ void swap4(float* v, int x) {
  const float a = x & 2 ? v[2] : v[0], b = x & 2 ? v[3] : v[1], c = x & 2 ? v[0] : v[2], d = x & 2 ? v[1] : v[3];
  v[0] = x & 1 ? b : a;
  v[1] = x & 1 ? a : b;
  v[2] = x & 1 ? d : c;
  v[3] = x & 1 ? c : d;
}

constexpr int kSelThreads = 128, kSelWarps = kSelThreads / 32;

// Where a thread stands: grid (chunk, b, group, tile), tile fastest.
//
// A thread holds a pair of channels (f2) and four states.  Its channel c is cl + (c ^ cx), its state s
// is 4 sg + (s ^ sx), where cx and sx come from its lane: lanes that exchange halves of their sums then
// keep the same registers and give the same ones away, and nothing has to be selected.  Swapped pairs
// are laid out as a second copy in shared memory.
//
// A warp lays out (and writes back) its own channels, W to a lane; the block shares B and C.
template <class T, int L, bool BWD>
struct SelThread {
  static constexpr int CG = 32 / L;            // pairs of channels in a warp
  static constexpr int CW = 2 * CG;            // channels of a warp
  static constexpr int CH = kSelWarps * CW;    // channels of a block
  static constexpr bool PARTS = BWD && L > 16; // the tiles may take several launches (see sel_shape)
  static constexpr int SP = 4 * L;             // padded states
  static constexpr int W = CW < 4 ? 2 : 4;     // channels that a lane lays out
  static constexpr int Q = CW / W;             // lanes to a row
  static constexpr int ROWS = 32 / Q;          // rows that a warp lays out at once
  static constexpr int NI = ROWS >= kSelSeg ? 1 : kSelSeg / ROWS;
  static constexpr int CC = L >= 2 ? 2 : 1;    // copies of the channels' arrays
  static constexpr int SC = BWD && CG >= 4 ? 2 : 1;   // copies of B and C
  static constexpr int CO = kSelSeg * CW + (CW < 32 ? CW : 0);   // where the second copy starts: in other banks
  static constexpr int AR = CC > 1 ? CO + kSelSeg * CW : kSelSeg * CW;   // a warp's array, in floats
  static constexpr int BO = kSelSeg * SP + (SP < 32 ? SP : 0);
  static constexpr int BC = SC > 1 ? BO + kSelSeg * SP : kSelSeg * SP;   // B or C, in floats
  using Raw = RawOf<T, W>;
  const SelArgs& p;
  int tid, lane, warp, sg, cl, cx, sx;
  int tile, g, b, chunk, n0, nn;               // first channel of the warp, channels of the warp there are
  int t0, t1, len;                             // the chunk's rows; rows of the sequence
  int col, row, left;                          // laying out: channels from col on of rows row, row + ROWS, ..
  int how;                                     // see sel_load
  __device__ __forceinline__ SelThread(const SelArgs& p_) : p(p_) {
    tid = threadIdx.x;
    lane = tid & 31;
    warp = tid >> 5;
    sg = lane % L;
    const int cg = lane / L;
    cl = cg * 2;
    cx = L >= 2 && sg & 1;
    sx = BWD ? (CG >= 2 && cg & 1 ? 2 : 0) | (CG >= 4 && cg & 2 ? 1 : 0) : 0;
    long long i = blockIdx.x;
    tile = (int)(i % p.tiles);
    i /= p.tiles;
    g = (int)(i % p.G);
    i /= p.G;
    b = (int)(i % p.B);
    chunk = (int)(i / p.B);
    const int c0 = ((PARTS ? p.tile0 : 0) + tile) * CH + warp * CW;
    n0 = g * p.Dg + c0;
    nn = max(0, min(CW, p.Dg - c0));
    t0 = chunk * p.steps;
    t1 = min(p.T, t0 + p.steps);
    len = row_length(p.lengths, p.wide, b, p.T);
    col = lane % Q * W;
    row = lane / Q;
    left = max(0, min(W, nn - col));
    how = p.vec == 4 && left == W ? 2 : p.vec >= 2;
  }
  // the thread's place in its row of the segment at t of a tensor (T,B,N)
  template <class E>
  __device__ __forceinline__ E* at(E* base, int t, long long st, long long sb) const {
    return base + (t + row) * st + b * sb + n0 + col;
  }
  // .. of B or C; the segment's rows are e / L of the thread's quads
  __device__ __forceinline__ const T* bc_at(const void* base, int t, long long st, long long sb) const {
    return (const T*)base + (t + tid / L) * st + b * sb + (long long)g * p.S + tid % L * 4;
  }
  // (.., N, S): register order.  One channel's four states are neighbours in memory; q points at
  // those of the thread's pair in their order there, and moves on by whole (B,N,S).
  __device__ __forceinline__ float* states_at(const float* base, size_t lead) const {
    return const_cast<float*>(base) + (lead * p.N + n0 + cl) * p.S + 4 * sg;
  }
  __device__ __forceinline__ void read_states(const float* q, bool four, f2* h) const {
    float v[2][4];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int s = 0; s < 4; ++s) v[c][s] = 0.f;
      if (four) {
        if (cl + c < nn && 4 * sg < p.S) *(float4*)v[c] = *(const float4*)(q + c * p.S);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
          if (cl + c < nn && 4 * sg + s < p.S) v[c][s] = q[c * p.S + s];
      }
      if (BWD) swap4(v[c], sx);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) h[s] = pair(cx ? v[1][s] : v[0][s], cx ? v[0][s] : v[1][s]);
  }
  __device__ __forceinline__ void write_states(float* q, bool four, const f2* h) const {
    float v[2][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float a, b;
      split(h[s], a, b);
      v[0][s] = cx ? b : a;
      v[1][s] = cx ? a : b;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (BWD) swap4(v[c], sx);
      if (four) {
        if (cl + c < nn && 4 * sg < p.S) *(float4*)(q + c * p.S) = f4(v[c]);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
          if (cl + c < nn && 4 * sg + s < p.S) q[c * p.S + s] = v[c][s];
      }
    }
  }
  __device__ __forceinline__ void load_state(const float* base, size_t lead, f2* h) const {
    if (base) {
      read_states(states_at(base, lead), p.S % 4 == 0 && !((uintptr_t)base & 15), h);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) h[s] = 0;
    }
  }
  __device__ __forceinline__ void load_decays(f2* A) const {
    load_state(p.A, 0, A);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float a, b;
      split(A[s], a, b);
      A[s] = pair(sel_finite(a), sel_finite(b));
    }
  }
  __device__ __forceinline__ void store_state(float* base, size_t lead, const f2* h) const {
    write_states(states_at(base, lead), p.S % 4 == 0, h);
  }
  __device__ __forceinline__ void load_weights(const float* w, float* v) const {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = w && i < left ? w[n0 + col + i] : 0.f;
  }
  // rows of B or C of a segment, 0 past the sequence's end and past S; a second copy with neighbours
  // swapped
  static constexpr int BCN = (kSelSeg * L + kSelThreads - 1) / kSelThreads;
  __device__ __forceinline__ void load_bc(const T* q, long long st, int seg, RawOf<T, 4>* v) const {
    constexpr int step = kSelThreads / L;
    const int n = p.S - tid % L * 4;
#pragma unroll
    for (int k = 0; k < BCN; ++k) {
      const int r = tid / L + k * step;
#pragma unroll
      for (unsigned i = 0; i < sizeof(v[k].w) / 4; ++i) v[k].w[i] = 0;
      if (n > 0 && r < kSelSeg && seg + r < len) sel_load<T, 4>(v[k], q + k * step * st, p.bcvec && n >= 4 ? 2 : 0, n);
    }
  }
  __device__ __forceinline__ void put_bc(const RawOf<T, 4>* v, float* dst) const {
#pragma unroll
    for (int k = 0; k < BCN; ++k) {
      const int e = tid + k * kSelThreads;
      if (e < kSelSeg * L) {
        float f[4];
        sel_floats<T, 4>(v[k], f);
        *(float4*)(dst + 4 * e) = f4(f);
        if (SC > 1) *(float4*)(dst + BO + 4 * e) = make_float4(f[1], f[0], f[3], f[2]);
      }
    }
  }
  __device__ __forceinline__ void get_bc(const float* src, int r, f2* v) const {
    const float* q = src + (SC > 1 && sx & 1 ? BO : 0) + r * SP + 4 * sg;
    float2 lo, hi;
    if (SC > 1) {
      lo = *(const float2*)(q + (sx & 2));
      hi = *(const float2*)(q + ((sx & 2) ^ 2));
    } else {
      const float4 f = *(const float4*)q;
      const bool up = BWD && sx & 2;
      lo = up ? make_float2(f.z, f.w) : make_float2(f.x, f.y);
      hi = up ? make_float2(f.x, f.y) : make_float2(f.z, f.w);
    }
    v[0] = pair(lo.x, lo.x); v[1] = pair(lo.y, lo.y); v[2] = pair(hi.x, hi.x); v[3] = pair(hi.y, hi.y);
  }
  // W channels of a row, and a copy with their pairs swapped
  __device__ __forceinline__ void put(float* dst, int r, const float* v) const {
    float* q = dst + r * CW + col;
    if constexpr (W == 4) {
      *(float4*)q = f4(v);
      if (CC > 1) *(float4*)(q + CO) = make_float4(v[1], v[0], v[3], v[2]);
    } else {
      *(float2*)q = make_float2(v[0], v[1]);
      if (CC > 1) *(float2*)(q + CO) = make_float2(v[1], v[0]);
    }
  }
  __device__ __forceinline__ void get(const float* src, int r, float* v) const {
    const float* q = src + r * CW + col;
    if constexpr (W == 4) *(float4*)v = *(const float4*)q;
    else *(float2*)v = *(const float2*)q;
  }
  __device__ __forceinline__ f2 get2(const float* src, int r) const {
    return *(const f2*)(src + (CC > 1 && cx ? CO : 0) + r * CW + cl);
  }
  // A pair's sums over the L lanes of its channels: afterwards v[0 .. NV) hold those of channels cl + cx, ..
  static constexpr int NV = L >= 2 ? 1 : 2;
  __device__ __forceinline__ void sum_states(f2 o, float* v) const {
    constexpr unsigned all = 0xffffffffu;
    split(o, v[0], v[1]);
    if (L >= 2) v[0] += __shfl_xor_sync(all, v[1], 1);
#pragma unroll
    for (int k = 2; k < L; k *= 2) v[0] += __shfl_xor_sync(all, v[0], k);
  }
  __device__ __forceinline__ bool owns() const { return L <= 2 || sg < 2; }
  // writes the sums to their channels of row r
  __device__ __forceinline__ void put_sums(float* dst, int r, const float* v) const {
    float* q = dst + r * CW + cl + cx;
#pragma unroll
    for (int i = 0; i < NV; ++i) q[i] = v[i];
  }
  // resets of a segment: bit r
  __device__ __forceinline__ uint32_t cuts(int seg, int end) const {
    return p.resets ? __ballot_sync(0xffffffffu, lane < kSelSeg && seg + lane < end && p.resets[(size_t)(seg + lane) * p.B + b]) : 0u;
  }
};

template <class T, int L, bool LOCAL>
constexpr int sel_fwd_smem() {
  using Th = SelThread<T, L, false>;
  return kSelWarps * (2 * Th::AR + kSelSeg * Th::CW) * 4 + 4 * Th::BC * 4;
}

// LOCAL: the chunk's map only (from a zero state), without C, the gate and y.  A segment's inputs
// are on their way while the one before is worked on; B and C have two places, so that the block
// meets once a segment.
template <class T, int L, bool LOCAL>
__global__ void __launch_bounds__(kSelThreads, L >= 4 ? 5 : 3) k_sel_fwd(const SelArgs p) {
  using Th = SelThread<T, L, false>;
  constexpr int ROWS = Th::ROWS, NI = Th::NI, W = Th::W;
  extern __shared__ float4 sm4[];
  const Th th(p);
  float* s_bc = (float*)sm4;                                          // [2][B, C]
  float* s_d = s_bc + 4 * Th::BC + th.warp * (2 * Th::AR + kSelSeg * Th::CW);
  float* s_x = s_d + Th::AR;
  float* s_o = s_x + Th::AR;
  const int end = min(th.t1, th.len);
  f2 A[4], h[4], sumd = 0;
  float bias[W], Dv[W];
  bool any_cut = false;
  th.load_decays(A);
  th.load_weights(p.bias, bias);
  th.load_weights(p.D, Dv);
  if (LOCAL) th.load_state(nullptr, 0, h);
  else if (p.chunks > 1) th.load_state(p.loc, (size_t)th.chunk * p.B + th.b, h);
  else th.load_state(p.h0, th.b, h);

  // pointers that move on with the segments
  const bool gate = !LOCAL && p.gate;
  const T *px = th.at((const T*)p.x, th.t0, p.x_t, p.x_b), *pz = th.at((const T*)p.dt, th.t0, p.dt_t, p.dt_b),
          *pu = gate ? th.at((const T*)p.gate, th.t0, p.u_t, p.u_b) : nullptr;
  const T *pB = th.bc_at(p.Bm, th.t0, p.bm_t, p.bm_b), *pC = th.bc_at(p.Cm, th.t0, p.cm_t, p.cm_b);
  T* py = th.at((T*)p.y, th.t0, p.y_t, p.y_b);
  float* pst = !LOCAL && p.states ? th.states_at(p.states, (size_t)(th.t0 / kSelSeg) * p.B + th.b) : nullptr;
  const bool four = p.S % 4 == 0;
  typename Th::Raw rx[NI], rz[NI], ru[NI], cx[NI], cu[NI];
  RawOf<T, 4> rB[Th::BCN], rC[Th::BCN];
  uint32_t rcut = 0;
  const auto fetch = [&](int seg) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = th.row + i * ROWS, t = seg + r;
      if (r < kSelSeg && t < end) {
        sel_load<T, W>(rx[i], px + i * ROWS * p.x_t, th.how, th.left);
        sel_load<T, W>(rz[i], pz + i * ROWS * p.dt_t, th.how, th.left);
        if (gate) sel_load<T, W>(ru[i], pu + i * ROWS * p.u_t, th.how, th.left);
      }
    }
    th.load_bc(pB, p.bm_t, seg, rB);
    if (!LOCAL) th.load_bc(pC, p.cm_t, seg, rC);
    rcut = th.cuts(seg, end);
    px += kSelSeg * p.x_t;
    pz += kSelSeg * p.dt_t;
    if (gate) pu += kSelSeg * p.u_t;
    pB += kSelSeg * p.bm_t;
    pC += kSelSeg * p.cm_t;
  };
  if (th.t0 < end) fetch(th.t0);
  int place = 0;
  for (int seg = th.t0; seg < end; seg += kSelSeg, place ^= 1) {
    const uint32_t cut = rcut;
    float *s_B = s_bc + place * 2 * Th::BC, *s_C = s_B + Th::BC;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = th.row + i * ROWS;
      if (r < kSelSeg) {   // past the end: delta 0 leaves a state as it is
        float dx[W] = {}, d[W] = {}, x[W], z[W], sig;
        if (seg + r < end) {
          sel_floats<T, W>(rx[i], x);
          sel_floats<T, W>(rz[i], z);
#pragma unroll
          for (int k = 0; k < W; ++k) {
            d[k] = k < th.left ? sel_delta<T, false>(z[k] + bias[k], p.softplus, sig) : 0.f;
            dx[k] = d[k] * x[k];
            d[k] *= kLog2e;
          }
        }
        th.put(s_d, r, d);
        th.put(s_x, r, dx);
      }
      cx[i] = rx[i];
      cu[i] = ru[i];
    }
    th.put_bc(rB, s_B);
    if (!LOCAL) th.put_bc(rC, s_C);
    __syncthreads();
    if (seg + kSelSeg < end) fetch(seg + kSelSeg);
    if (pst) {
      th.write_states(pst, four, h);
      pst += (size_t)p.B * p.N * p.S;
    }
    any_cut |= cut != 0;
    const auto step = [&](int r) {
      f2 Bv[4], Cv[4];
      const f2 d = th.get2(s_d, r), dx = th.get2(s_x, r);
      th.get_bc(s_B, r, Bv);
#pragma unroll
      for (int s = 0; s < 4; ++s) h[s] = fma2(sel_decay2(d, A[s]), h[s], mul2(dx, Bv[s]));
      if (LOCAL) {
        sumd = fma2(d, pair(1.f, 1.f), sumd);
      } else {
        th.get_bc(s_C, r, Cv);
        f2 o2 = mul2(Cv[0], h[0]);
#pragma unroll
        for (int s = 1; s < 4; ++s) o2 = fma2(Cv[s], h[s], o2);
        float o[2];
        th.sum_states(o2, o);
        if (th.owns()) th.put_sums(s_o, r, o);
      }
    };
    if (!cut) {            // steps without a branch between them
#pragma unroll
      for (int r = 0; r < kSelSeg; ++r) step(r);
    } else {
#pragma unroll 1
      for (int r = 0; r < kSelSeg; ++r) {
        if (cut >> r & 1) {
#pragma unroll
          for (int s = 0; s < 4; ++s) h[s] = 0;
        }
        step(r);
      }
    }
    __syncwarp();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = th.row + i * ROWS, t = seg + r;
        if (r < kSelSeg && t < end) {
          float o[W], x[W];
          th.get(s_o, r, o);
          sel_floats<T, W>(cx[i], x);
#pragma unroll
          for (int k = 0; k < W; ++k) o[k] = fmaf(Dv[k], x[k], o[k]);
          if (gate) {
            float u[W], sg, so;
            sel_floats<T, W>(cu[i], u);
#pragma unroll
            for (int k = 0; k < W; ++k) {
              sigmoid_pair<false>(u[k], sg, so);
              o[k] *= u[k] * sg;
            }
          }
          sel_store<T, W>(py + i * ROWS * p.y_t, th.how, th.left, o);
        }
      }
      py += kSelSeg * p.y_t;
      __syncwarp();
    }
  }
  if (LOCAL) {
    const size_t lead = (size_t)th.chunk * p.B + th.b;
    th.store_state(p.loc, lead, h);
    if (th.sg == 0) {   // cx = 0
      float s[2];
      split(sumd, s[0], s[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (th.cl + c < th.nn) p.sumd[lead * p.N + th.n0 + th.cl + c] = s[c];
    }
    if (th.tid == 0 && th.tile == 0 && th.g == 0) p.cut[lead] = any_cut;
    return;
  }
  const float zero[W] = {};
  for (int t = max(th.t0, end) + th.row; t < th.t1; t += ROWS) sel_store<T, W>(th.at((T*)p.y, t - th.row, p.y_t, p.y_b), th.how, th.left, zero);
  if (th.chunk == max(th.len - 1, 0) / p.steps) th.store_state(p.hT, th.b, h);
}

// The states (BACK: the gradients of the states) in front of (behind) each chunk, in place of its
// own share: one thread per (b, n, s), in time order.  start: h0 or ghT.
template <bool BACK>
__global__ void __launch_bounds__(64) k_sel_join(const SelArgs p, const float* __restrict__ start) {
  const size_t row = (size_t)p.N * p.S, all = row * p.B;
  const size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  if (i >= all) return;
  const int b = (int)(i / row);
  const size_t ns = i - b * row, n = ns / p.S;
  const float A = sel_finite(p.A[ns]);
  float h = start ? start[i] : 0.f;
  constexpr int U = 16;                 // chunks whose maps are on their way together
  for (int c0 = 0; c0 < p.chunks; c0 += U) {
    float loc[U], d[U];
    uint8_t cut[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int c = c0 + k < p.chunks ? (BACK ? p.chunks - 1 - (c0 + k) : c0 + k) : 0;
      const size_t lead = (size_t)c * p.B + b;
      loc[k] = p.loc[lead * row + ns];
      d[k] = p.sumd[lead * p.N + n];
      cut[k] = p.cut[lead];
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int c = BACK ? p.chunks - 1 - (c0 + k) : c0 + k;
      if (c0 + k < p.chunks) {
        p.loc[((size_t)c * p.B + b) * row + ns] = h;
        // (0 stays 0 also where a chunk grows past the largest float)
        h = cut[k] || h == 0.f ? loc[k] : fmaf(sel_exp2(A * d[k]), h, loc[k]);
      }
    }
  }
}

// places of the channels' sums of dB and dC: two, so that the block meets once a segment, unless they are large
template <int L>
constexpr int sel_reds() { return L >= 16 ? 1 : 2; }
template <class T, int L, bool LOCAL>
constexpr int sel_bwd_smem() {
  using Th = SelThread<T, L, true>;
  return kSelWarps * (LOCAL ? 2 : 3) * Th::AR * 4 + (LOCAL ? 2 : 4) * Th::BC * 4 +
         (LOCAL ? 0 : sel_reds<L>() * kSelWarps * kSelSeg * 2 * Th::SP * 4 + (kSelSeg - 1) * 32 * kSelThreads);
}

// LOCAL: the chunk's share of the states' gradients only (from a zero gradient behind it)
template <class T, int L, bool LOCAL>
__global__ void __launch_bounds__(kSelThreads, L == 4 || L == 8 ? 3 : 2) k_sel_bwd(const SelArgs p) {
  using Th = SelThread<T, L, true>;
  constexpr int SP = Th::SP, ROWS = Th::ROWS, NI = Th::NI, W = Th::W, CG = Th::CG, AR = Th::AR, BC = Th::BC;
  constexpr int nt = kSelThreads, REDS = sel_reds<L>(), RED = kSelWarps * kSelSeg * 2 * SP;
  extern __shared__ float4 sm4[];
  const Th th(p);
  ulonglong2* hist = (ulonglong2*)sm4;                           // [1 .. kSelSeg)[2][nt]: the state before each step
  float* s_bc = (float*)(LOCAL ? hist : hist + (kSelSeg - 1) * 2 * nt);   // [2][C, B]
  float* s_red = s_bc + (LOCAL ? 2 : 4) * BC;          // [REDS][warp][kSelSeg][2 SP]
  float* s_d = (LOCAL ? s_red : s_red + REDS * RED) + th.warp * (LOCAL ? 2 : 3) * AR;   // later the sums for ddt
  float* s_go = s_d + AR;                                        // gy silu(gate); later sum C h
  float* s_x = s_go + AR;                                        // later sum G B; not in a LOCAL pass
  const int end = min(th.t1, th.len);
  const size_t lead = (size_t)th.chunk * p.B + th.b;
  f2 A[4], G[4], dA[4], sumd = 0;
  float bias[W], Dv[W], dD[W] = {}, db[W] = {};
  bool any_cut = false;
  th.load_decays(A);
  th.load_weights(p.bias, bias);
  th.load_weights(p.D, Dv);
#pragma unroll
  for (int s = 0; s < 4; ++s) dA[s] = 0;
  if (LOCAL) th.load_state(nullptr, 0, G);
  else if (p.chunks > 1) th.load_state(p.loc, lead, G);
  else th.load_state(p.ghT, th.b, G);

  const int segs = end > th.t0 ? (end - th.t0 + kSelSeg - 1) / kSelSeg : 0;
  // pointers that move back with the segments
  const int tl = th.t0 + max(segs - 1, 0) * kSelSeg;
  const bool gate = p.gate, grad = p.gy;
  const T *px = th.at((const T*)p.x, tl, p.x_t, p.x_b), *pz = th.at((const T*)p.dt, tl, p.dt_t, p.dt_b),
          *pu = th.at((const T*)p.gate, tl, p.u_t, p.u_b), *pg = th.at((const T*)p.gy, tl, p.gy_t, p.gy_b);
  const T *pB = th.bc_at(p.Bm, tl, p.bm_t, p.bm_b), *pC = th.bc_at(p.Cm, tl, p.cm_t, p.cm_b);
  T *pdx = th.at((T*)p.dx, tl, p.dx_t, p.dx_b), *pdz = th.at((T*)p.ddt, tl, p.ddt_t, p.ddt_b),
    *pdu = th.at((T*)p.dgate, tl, p.du_t, p.du_b);
  const float* pst = LOCAL ? nullptr : th.states_at(p.states, (size_t)(tl / kSelSeg) * p.B + th.b);
  const bool four = p.S % 4 == 0 && !((uintptr_t)p.states & 15);
  if (!LOCAL) {   // rows past the end: zero gradients
    const float zero[W] = {};
    for (int t = max(th.t0, end) + th.row; t < th.t1; t += ROWS) {
      if (p.dx) sel_store<T, W>(th.at((T*)p.dx, t - th.row, p.dx_t, p.dx_b), th.how, th.left, zero);
      if (p.ddt) sel_store<T, W>(th.at((T*)p.ddt, t - th.row, p.ddt_t, p.ddt_b), th.how, th.left, zero);
      if (p.dgate) sel_store<T, W>(th.at((T*)p.dgate, t - th.row, p.du_t, p.du_b), th.how, th.left, zero);
    }
  }
  // dB and dC of all rows of the chunk are written, zeros past the end
  const long long bc_t = (long long)p.B * p.G * p.S, bc_0 = ((long long)th.tile * p.T * p.B + th.b) * p.G * p.S + (long long)th.g * p.S;
  const auto write_bc = [&](int seg, const float* red) {
#pragma unroll
    for (int e0 = 0; e0 < kSelSeg * 2 * SP; e0 += nt) {
      const int e = e0 + th.tid, r = e / (2 * SP), q = e % (2 * SP), s = q % SP, t = seg + r;
      if (e < kSelSeg * 2 * SP && s < p.S && t < th.t1) {
        float v = 0.f;
        if (t < end)
#pragma unroll
          for (int w = 0; w < kSelWarps; ++w) v += red[w * kSelSeg * 2 * SP + e];
        float* dst = q < SP ? p.dB : p.dC;
        if (dst) {
          dst += bc_0 + t * bc_t + s;
          // one block adds to a place in a launch: no order of atomics, and no wait for what is there (T=250 B=32
          // N=2048 S=128 in three launches 5461 us, with a read 9742)
          if (Th::PARTS && p.add) atomicAdd(dst, v);
          else *dst = v;
        }
      }
    }
  };
  const bool bc = !LOCAL && (p.dB || p.dC);
  if (bc)
    for (int seg = th.t0 + segs * kSelSeg; seg < th.t1; seg += kSelSeg) write_bc(seg, s_red);

  typename Th::Raw rx[NI], rz[NI], ru[NI], rg[NI];
  RawOf<T, 4> rB[Th::BCN], rC[Th::BCN];
  uint32_t rcut = 0;
  f2 h[4];
  const auto fetch = [&](int seg) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = th.row + i * ROWS, t = seg + r;
      if (r < kSelSeg && t < end) {
        if (!LOCAL) sel_load<T, W>(rx[i], px + i * ROWS * p.x_t, th.how, th.left);
        sel_load<T, W>(rz[i], pz + i * ROWS * p.dt_t, th.how, th.left);
        if (gate) sel_load<T, W>(ru[i], pu + i * ROWS * p.u_t, th.how, th.left);
        if (grad) sel_load<T, W>(rg[i], pg + i * ROWS * p.gy_t, th.how, th.left);
      }
    }
    th.load_bc(pC, p.cm_t, seg, rC);
    if (!LOCAL) {
      th.load_bc(pB, p.bm_t, seg, rB);
      th.read_states(pst, four, h);
      px -= kSelSeg * p.x_t;
      pB -= kSelSeg * p.bm_t;
      pst -= (size_t)p.B * p.N * p.S;
    }
    rcut = th.cuts(seg, end);
    pz -= kSelSeg * p.dt_t;
    pu -= kSelSeg * p.u_t;
    pg -= kSelSeg * p.gy_t;
    pC -= kSelSeg * p.cm_t;
  };
  if (segs > 0) fetch(th.t0 + (segs - 1) * kSelSeg);
  int place = 0;
  for (int k = segs - 1; k >= 0; --k, place ^= 1) {
    const int seg = th.t0 + k * kSelSeg;
    const uint32_t cut = rcut;
    float *s_C = s_bc + place * (LOCAL ? 1 : 2) * BC, *s_B = s_C + BC;
    float* red = s_red + (REDS > 1 ? place * RED : 0);
    float x[NI][W], d[NI][W], sig[NI][W], go[NI][W], gs[NI][W];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = th.row + i * ROWS;
#pragma unroll
      for (int q = 0; q < W; ++q) x[i][q] = d[i][q] = sig[i][q] = go[i][q] = gs[i][q] = 0.f;
      if (r < kSelSeg) {
        if (seg + r < end) {
          float z[W], u[W];
          if (!LOCAL) sel_floats<T, W>(rx[i], x[i]);
          sel_floats<T, W>(rz[i], z);
          if (grad) sel_floats<T, W>(rg[i], go[i]);
#pragma unroll
          for (int q = 0; q < W; ++q) d[i][q] = q < th.left ? sel_delta<T, !LOCAL>(z[q] + bias[q], p.softplus, sig[i][q]) : 0.f;
          if (gate) {
            sel_floats<T, W>(ru[i], u);
#pragma unroll
            for (int q = 0; q < W; ++q) {
              float sg, so;
              sigmoid_pair<false>(u[q], sg, so);
              gs[i][q] = go[i][q] * (sg * fmaf(u[q], so, 1.f));
              go[i][q] *= u[q] * sg;
            }
          }
        }
        float d2[W], dx[W];
#pragma unroll
        for (int q = 0; q < W; ++q) {
          d2[q] = d[i][q] * kLog2e;
          dx[q] = d[i][q] * x[i][q];
        }
        th.put(s_d, r, d2);
        th.put(s_go, r, go[i]);
        if (!LOCAL) th.put(s_x, r, dx);
      }
    }
    th.put_bc(rC, s_C);
    if (!LOCAL) th.put_bc(rB, s_B);
    __syncthreads();
    if (bc && k + 1 < segs) {
      write_bc(seg + kSelSeg, s_red + (REDS > 1 ? (place ^ 1) * RED : 0));
      if (REDS == 1) __syncthreads();
    }
    f2 first[4] = {};
    if (!LOCAL) {
#pragma unroll
      for (int s = 0; s < 4; ++s) first[s] = h[s];
      const auto step = [&](int r) {
        f2 Bv[4];
        const f2 dd = th.get2(s_d, r), dx = th.get2(s_x, r);
        th.get_bc(s_B, r, Bv);
#pragma unroll
        for (int s = 0; s < 4; ++s) h[s] = fma2(sel_decay2(dd, A[s]), h[s], mul2(dx, Bv[s]));
        if (r + 1 < kSelSeg) {
          hist[r * 2 * nt + th.tid] = make_ulonglong2(h[0], h[1]);
          hist[(r * 2 + 1) * nt + th.tid] = make_ulonglong2(h[2], h[3]);
        }
      };
      if (!cut) {          // steps without a branch between them
#pragma unroll
        for (int r = 0; r < kSelSeg; ++r) step(r);
      } else {
#pragma unroll 1
        for (int r = 0; r < kSelSeg; ++r) {
          if (cut >> r & 1) {
#pragma unroll
            for (int s = 0; s < 4; ++s) h[s] = 0;
          }
          step(r);
        }
      }
    }
    any_cut |= cut != 0;
    // one step back from pre, the state before it; nothing passes a reset, an infinite state neither
    const auto back = [&](int r, const f2* pre, bool here) {
      f2 Cv[4];
      const f2 dd = th.get2(s_d, r), gg = th.get2(s_go, r);
      th.get_bc(s_C, r, Cv);
      if constexpr (LOCAL) {
        sumd = fma2(dd, pair(1.f, 1.f), sumd);
#pragma unroll
        for (int s = 0; s < 4; ++s) G[s] = mul2(sel_decay2(dd, A[s]), fma2(Cv[s], gg, G[s]));
        if (here) {
#pragma unroll
          for (int s = 0; s < 4; ++s) G[s] = 0;
        }
      } else {
        f2 Bv[4], ag[4], w[4], bB[4], bC[4], gb2, wa2, o2;
        const f2 dx = th.get2(s_x, r);
        th.get_bc(s_B, r, Bv);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const f2 Gt = fma2(Cv[s], gg, G[s]);
          o2 = s ? fma2(Cv[s], h[s], o2) : mul2(Cv[s], h[s]);
          bC[s] = mul2(gg, h[s]);
          bB[s] = mul2(Gt, dx);
          gb2 = s ? fma2(Gt, Bv[s], gb2) : mul2(Gt, Bv[s]);
          ag[s] = mul2(sel_decay2(dd, A[s]), Gt);
          w[s] = mul2(ag[s], pre[s]);
          h[s] = pre[s];
        }
        if (here) {
#pragma unroll
          for (int s = 0; s < 4; ++s) ag[s] = w[s] = 0;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          wa2 = s ? fma2(w[s], A[s], wa2) : mul2(w[s], A[s]);
          dA[s] = fma2(w[s], dd, dA[s]);
          G[s] = ag[s];
        }
        float vB[4], vC[4], gb[2], wa[2], o[2];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          float a, b;
          split(bB[s], a, b);
          vB[s] = a + b;
          split(bC[s], a, b);
          vC[s] = a + b;
        }
        th.sum_states(gb2, gb);
        th.sum_states(wa2, wa);
        th.sum_states(o2, o);
        __syncwarp();         // every lane has read its row
        if (th.owns()) {
          th.put_sums(s_x, r, gb);
          th.put_sums(s_d, r, wa);
          th.put_sums(s_go, r, o);
        }
        // over the channels: lanes L, 2 L, .. apart; at last one of two lanes keeps dB, the other dC
        constexpr unsigned all = 0xffffffffu;
        if (CG >= 2) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            vB[s] += __shfl_xor_sync(all, vB[s + 2], L);
            vC[s] += __shfl_xor_sync(all, vC[s + 2], L);
          }
        }
        if (CG >= 4) {
          vB[0] += __shfl_xor_sync(all, vB[1], 2 * L);
          vC[0] += __shfl_xor_sync(all, vC[1], 2 * L);
        }
        float* q = red + (th.warp * kSelSeg + r) * 2 * SP + 4 * th.sg + th.sx;
        if constexpr (CG >= 8) {
          const bool up = th.lane & (4 * L);
          float v = (up ? vC[0] : vB[0]) + __shfl_xor_sync(all, up ? vB[0] : vC[0], 4 * L);
#pragma unroll
          for (int i = 8 * L; i < 32; i *= 2) v += __shfl_xor_sync(all, v, i);
          if (th.lane < 8 * L) q[up ? SP : 0] = v;
        } else {
          constexpr int n = CG >= 4 ? 1 : CG >= 2 ? 2 : 4;
#pragma unroll
          for (int s = 0; s < n; ++s) {
            q[s] = vB[s];
            q[SP + s] = vC[s];
          }
        }
      }
    };
    const auto before = [&](int r, f2* pre) {
      if (!LOCAL) {
        const ulonglong2 q0 = hist[(r - 1) * 2 * nt + th.tid], q1 = hist[(r * 2 - 1) * nt + th.tid];
        pre[0] = q0.x; pre[1] = q0.y; pre[2] = q1.x; pre[3] = q1.y;
      }
    };
    f2 pre[4];
    if (!cut) {
#pragma unroll 7
      for (int r = kSelSeg - 1; r > 0; --r) {
        before(r, pre);
        back(r, pre, false);
      }
    } else {
#pragma unroll 1
      for (int r = kSelSeg - 1; r > 0; --r) {
        before(r, pre);
        back(r, pre, cut >> r & 1);
      }
    }
    back(0, first, cut & 1);
    if (k > 0) fetch(seg - kSelSeg);
    __syncwarp();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = th.row + i * ROWS, t = seg + r;
        if (r < kSelSeg && t < end) {
          float gb[W], wa[W], o[W], vx[W], vz[W], vu[W];
          th.get(s_x, r, gb);
          th.get(s_d, r, wa);
          th.get(s_go, r, o);
#pragma unroll
          for (int q = 0; q < W; ++q) {
            vx[q] = fmaf(gb[q], d[i][q], Dv[q] * go[i][q]);
            vz[q] = fmaf(gb[q], x[i][q], wa[q]) * sig[i][q];
            vu[q] = gs[i][q] * fmaf(Dv[q], x[i][q], o[q]);
            dD[q] = fmaf(go[i][q], x[i][q], dD[q]);
            db[q] += vz[q];
          }
          if (p.dx) sel_store<T, W>(pdx + i * ROWS * p.dx_t, th.how, th.left, vx);
          if (p.ddt) sel_store<T, W>(pdz + i * ROWS * p.ddt_t, th.how, th.left, vz);
          if (p.dgate) sel_store<T, W>(pdu + i * ROWS * p.du_t, th.how, th.left, vu);
        }
      }
      pdx -= kSelSeg * p.dx_t;
      pdz -= kSelSeg * p.ddt_t;
      pdu -= kSelSeg * p.du_t;
      __syncwarp();
    }
  }
  if (bc && segs > 0) {
    __syncthreads();
    write_bc(th.t0, s_red + (REDS > 1 ? (place ^ 1) * RED : 0));
  }
  if (LOCAL) {
    th.store_state(p.loc, lead, G);
    if (th.sg == 0) {
      float s[2];
      split(sumd, s[0], s[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (th.cl + c < th.nn) p.sumd[lead * p.N + th.n0 + th.cl + c] = s[c];
    }
    if (th.tid == 0 && th.tile == 0 && th.g == 0) p.cut[lead] = any_cut;
    return;
  }
  if (p.dh0 && th.chunk == 0) th.store_state(p.dh0, th.b, G);
  if (p.dA) {
    const f2 ln2 = pair(kLn2, kLn2);
#pragma unroll
    for (int s = 0; s < 4; ++s) dA[s] = mul2(dA[s], ln2);
    th.store_state(p.dA, lead, dA);
  }
  // dD and db: over the lanes that have laid out the same channels
#pragma unroll
  for (int q = 0; q < W; ++q) {
#pragma unroll
    for (int i = Th::Q; i < 32; i *= 2) {
      dD[q] += __shfl_xor_sync(0xffffffffu, dD[q], i);
      db[q] += __shfl_xor_sync(0xffffffffu, db[q], i);
    }
    if (th.row == 0 && q < th.left) {
      const size_t e = lead * p.N + th.n0 + th.col + q;
      if (p.dD) p.dD[e] = dD[q];
      if (p.db) p.db[e] = db[q];
    }
  }
}

// out[j] = sum over parts of part[k][j], in order and in 64 bits.  Block: 32 columns by 32 runs of parts.
static __global__ void __launch_bounds__(1024) k_sel_sum(long long cols, long long parts, const float* __restrict__ part,
                                                  float* __restrict__ out) {
  __shared__ double sum[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const long long j = blockIdx.x * 32LL + lane;
  const long long p0 = parts * run / 32, p1 = parts * (run + 1) / 32;
  double s = 0.0;
  if (j < cols)
    for (long long q = p0; q < p1; ++q) s += part[q * cols + j];
  sum[run][lane] = s;
  __syncthreads();
  if (run == 0 && j < cols) {
    double t = 0.0;
    for (int r = 0; r < 32; ++r) t += sum[r][lane];
    out[j] = (float)t;
  }
}
// dB and dC (T,B,G,S) from their partial sums, one to a tile of channels of a launch
template <class T>
__global__ void __launch_bounds__(256) k_sel_bc(long long cols, int tiles, const float* __restrict__ dB,
                                                const float* __restrict__ dC, T* __restrict__ oB, T* __restrict__ oC) {
  const long long j = blockIdx.x * 256LL + threadIdx.x;
  if (j >= cols) return;
  if (oB) {
    float s = 0.f;
    for (int k = 0; k < tiles; ++k) s += dB[k * cols + j];
    oB[j] = from_f<T>(s);
  }
  if (oC) {
    float s = 0.f;
    for (int k = 0; k < tiles; ++k) s += dC[k * cols + j];
    oC[j] = from_f<T>(s);
  }
}

// One time step: L lanes to a channel, four states a lane, everything that a lane reads on its way at once.
// state and next (B,N,S) may be one tensor.
struct SelStep {
  int B, N, S, G, Dg, softplus;
  int four, bcvec;                  // four: states in 16-byte accesses; bcvec: B and C in fours
  const void *x, *dt, *Bm, *Cm, *gate;
  const float *A, *D, *bias;
  const float* state;
  const uint8_t* active;
  void* y;
  float* next;
  long long x_b, dt_b, u_b, bm_b, cm_b;
};
// What a lane reads of a sequence besides its states, and what it makes of them.  Its quads of states are
// 4 L apart, so that the lanes of a channel read whole sectors.
template <class T, int L, int Q>
struct SelLane {
  float A[Q], Bv[Q], Cv[Q], x, z, u, D, bias;
  const SelStep& p;
  int n, g, s0;
  __device__ __forceinline__ SelLane(const SelStep& p_, int n_, int s0_) : p(p_), n(n_), s0(s0_) {
    g = p.G == 1 ? 0 : (unsigned)n / (unsigned)p.Dg;
  }
  static constexpr int off(int s) { return s / 4 * 4 * L + s % 4; }
  __device__ __forceinline__ void weights(bool on) {
    const float* Ap = p.A + (size_t)n * p.S + s0;
#pragma unroll
    for (int s = 0; s < Q; ++s) A[s] = on && s0 + off(s) < p.S ? sel_finite(Ap[off(s)]) : 0.f;
    D = on && p.D ? p.D[n] : 0.f;
    bias = on && p.bias ? p.bias[n] : 0.f;
  }
  __device__ __forceinline__ void inputs(bool act, long long b) {
    x = z = u = 0.f;
#pragma unroll
    for (int s = 0; s < Q; ++s) Bv[s] = Cv[s] = 0.f;
    if (!act) return;            // what does not count is not read
    x = to_f(((const T*)p.x)[b * p.x_b + n]);
    z = to_f(((const T*)p.dt)[b * p.dt_b + n]);
    if (p.gate) u = to_f(((const T*)p.gate)[b * p.u_b + n]);
    const T *Bp = (const T*)p.Bm + b * p.bm_b + (long long)g * p.S + s0, *Cp = (const T*)p.Cm + b * p.cm_b + (long long)g * p.S + s0;
#pragma unroll
    for (int k = 0; k < Q; k += 4) {
      if (p.bcvec) {
        if (s0 + off(k) < p.S) {
          unpack_vec<T, 4>(*(const VecOf<T, 4>*)(Bp + off(k)), Bv + k);
          unpack_vec<T, 4>(*(const VecOf<T, 4>*)(Cp + off(k)), Cv + k);
        }
      } else {
#pragma unroll
        for (int s = k; s < k + 4; ++s)
          if (s0 + off(s) < p.S) {
            Bv[s] = to_f(Bp[off(s)]);
            Cv[s] = to_f(Cp[off(s)]);
          }
      }
    }
  }
  __device__ __forceinline__ void load(const float* at, float* h) const {
#pragma unroll
    for (int k = 0; k < Q; k += 4) {
      if (p.four) {
        if (s0 + off(k) < p.S) unpack_vec<float, 4>(*(const VecOf<float, 4>*)(at + off(k)), h + k);
      } else {
#pragma unroll
        for (int s = k; s < k + 4; ++s)
          if (s0 + off(s) < p.S) h[s] = at[off(s)];
      }
    }
  }
  // h <- the next states, written to `at`; the output to y
  __device__ __forceinline__ void run(bool on, bool act, float* h, float* at, T* y) {
    float sig, o = 0.f;
    const float d = sel_delta<T, false>(z + bias, p.softplus, sig), e = d * kLog2e, dx = d * x;
    if (act) {
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        h[s] = fmaf(sel_exp2(fmaf(e, A[s], kSelLow)), h[s], dx * Bv[s]);
        o = fmaf(Cv[s], h[s], o);
      }
    }
    if (on) {
#pragma unroll
      for (int k = 0; k < Q; k += 4) {
        if (p.four) {
          if (s0 + off(k) < p.S) *(float4*)(at + off(k)) = f4(h + k);
        } else {
#pragma unroll
          for (int s = k; s < k + 4; ++s)
            if (s0 + off(s) < p.S) at[off(s)] = h[s];
        }
      }
    }
#pragma unroll
    for (int j = 1; j < L; j *= 2) o += __shfl_xor_sync(0xffffffffu, o, j);
    if (on && s0 == 0) {
      float v = fmaf(D, x, o);
      if (p.gate) {
        float s, so;
        sigmoid_pair<false>(u, s, so);
        v *= u * s;
      }
      *y = from_f<T>(act ? v : 0.f);
    }
  }
};
template <class T, int L>
__global__ void __launch_bounds__(256) k_sel_step(const SelStep p) {
  const long long i = blockIdx.x * 256LL + threadIdx.x, at = i / L;
  const bool on = at < (long long)p.B * p.N;
  const unsigned ch = on ? (unsigned)at : 0u;           // B N fits 31 bits
  const int b = (int)(ch / (unsigned)p.N);
  const bool act = on && (!p.active || p.active[b]);
  SelLane<T, L, 4> t(p, (int)(ch - (unsigned)b * p.N), 4 * (int)(i % L));
  const long long s = (long long)ch * p.S + t.s0;
  float h[4] = {};
  if (on && p.state) t.load(p.state + s, h);
  t.inputs(act, b);
  t.weights(act);
  t.run(on, act, h, p.next + s, (T*)p.y + ch);
}

// The same where there are more sequences than threads: a lane (Q states) keeps its channel's weights and
// takes every `rows`-th sequence, whose states are on their way to its own place in shared memory while it
// works on the ones before (a lane per sequence has too few bytes in flight: 4096 x 512 x 16 states bf16 in
// a graph 88 -> 61 us, 2048 x 700 x 24 fp32 120 -> 69, of 41 that the states take).
constexpr int kSelStages = 3;
__device__ __forceinline__ void cp_async16(void* smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <class T, int L, int Q>
__global__ void __launch_bounds__(256, 4) k_sel_steps(const SelStep p, int rows) {
  __shared__ float4 ring[kSelStages][Q / 4][256];
  const long long i = blockIdx.x * 256LL + threadIdx.x, NL = (long long)p.N * L;
  const bool there = i < NL * rows;
  long long b = i / NL;
  SelLane<T, L, Q> t(p, (int)(i % NL / L), 4 * (int)(i % L));
  t.weights(there);
  const auto place = [&](long long row) { return (row * p.N + t.n) * p.S + t.s0; };
  const auto fetch = [&](int stage, long long row) {
    if (there && row < p.B) {
#pragma unroll
      for (int k = 0; k < Q / 4; ++k)
        if (t.s0 + 4 * L * k < p.S) cp_async16(&ring[stage][k][threadIdx.x], p.state + place(row) + 4 * L * k);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kSelStages; ++j) fetch(j, b + (long long)j * rows);
  int stage = 0;
  for (int k = 0; k < p.B; k += min(rows, p.B - k), b += rows) {   // the same number of rounds in a whole warp
    const bool on = there && b < p.B;
    const bool act = on && (!p.active || p.active[b]);
    t.inputs(act, b);
    cp_async_wait<kSelStages - 1>();
    float h[Q] = {};
#pragma unroll
    for (int q = 0; q < Q / 4; ++q)
      if (t.s0 + 4 * L * q < p.S) unpack_vec<float, 4>(*(const VecOf<float, 4>*)&ring[stage][q][threadIdx.x], h + 4 * q);
    t.run(on, act, h, p.next + place(b), (T*)p.y + b * p.N + t.n);
    fetch(stage, b + (long long)kSelStages * rows);
    stage = stage + 1 == kSelStages ? 0 : stage + 1;
  }
}

}  // namespace delrec
