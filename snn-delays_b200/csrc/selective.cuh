// Selective state space scan and its gradients.  Per channel n of group g and state s:
//
//   delta_t = softplus(dt_t + dt_bias)                      (or dt_t + dt_bias)
//   h_t[s]  = exp(delta_t A[s]) h_{t-1}[s] + delta_t B_t[s] x_t
//   y_t     = (sum_s C_t[s] h_t[s] + D x_t) silu(gate_t)
//
// A thread holds 4 channels x 4 states; L lanes (4 L >= S) share a channel's states, the other
// 32 / L lane groups of a warp hold other channels.  So B_t and C_t are four values a thread, the
// sums over states (y, dx, ddt) run over four values in the thread and then over L lanes, and those over
// channels (dB, dC) over four values and then over 32 / L lanes: either way a
// lane hands on half of what it holds at each exchange.  A block walks kSelSeg steps at a time, whose
// inputs it lays out in shared memory in float32; states stay in registers.
//
// The backward pass keeps the states before every kSelSeg-th step (written by the forward pass),
// recomputes those in between into shared memory and walks the segment back.  Where the rows are
// few, time is cut into chunks: their affine maps come first (k_sel_local; the product of a chunk's
// decays is exp(A sum delta)), are joined in time order (k_sel_join), and then every chunk runs from
// its own start.
//
// What bounds it: the exponentials, 16 a clock and SM (one a state forward, two backward), with the
// issue slots close behind.  Sums and states are float32.
#pragma once

#include "seq_common.cuh"

namespace delrec {

constexpr int kSelSeg = 8;       // steps of a segment; distance of the states kept for the backward pass
constexpr int kSelMaxS = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct SelArgs {
  int T, B, N, S, G, Dg;          // Dg = N / G channels to a group
  int softplus, wide, vec;        // vec: rows of x, dt, gate, y and their gradients in fours
  int chunks, steps, tiles, CH;   // chunks of `steps` rows; tiles of CH channels to a group
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
  float *dB, *dC;                 // (tiles, T, B, G, S): partial sums
  long long gy_t, gy_b, dx_t, dx_b, ddt_t, ddt_b, du_t, du_b;
};

__device__ __forceinline__ float sel_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Sum of v[0..NV) over the lanes that differ in the bits FIRST, 2 FIRST, .. < LAST of the lane: at
// each exchange a lane keeps half of the values.  Afterwards v[0 .. max(1, NV / lanes)) hold the
// sums of the values from sel_owner on.
template <int FIRST, int LAST, int NV>
__device__ __forceinline__ void sel_sum(float* v, int lane) {
  if constexpr (FIRST < LAST) {
    if constexpr (NV > 1) {
      constexpr int H = NV / 2;
      const bool up = lane & FIRST;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float keep = up ? v[i + H] : v[i], give = up ? v[i] : v[i + H];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, FIRST);
      }
      sel_sum<2 * FIRST, LAST, H>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], FIRST);
      sel_sum<2 * FIRST, LAST, 1>(v, lane);
    }
  }
}
template <int FIRST, int LAST, int NV>
__device__ __forceinline__ int sel_owner(int lane) {
  if constexpr (FIRST < LAST && NV > 1) return (lane & FIRST ? NV / 2 : 0) + sel_owner<2 * FIRST, LAST, NV / 2>(lane);
  return 0;
}
// the first of the lanes that hold the same sums
template <int FIRST, int LAST, int NV>
__device__ __forceinline__ bool sel_first(int lane) {
  if constexpr (FIRST < LAST) {
    if constexpr (NV > 1) return sel_first<2 * FIRST, LAST, NV / 2>(lane);
    else return !(lane & FIRST) && sel_first<2 * FIRST, LAST, 1>(lane);
  }
  return true;
}

// delta and its derivative by dt
__device__ __forceinline__ float sel_delta(float z, int softplus, float& d) {
  if (!softplus) {
    d = 1.f;
    return z;
  }
  const float t = expf(-fabsf(z)), r = 1.f / (1.f + t);
  d = z >= 0.f ? r : t * r;
  return fmaxf(z, 0.f) + log1pf(t);
}

template <class T>
__device__ __forceinline__ void sel_load4(const void* base, long long at, bool vec, int left, float* v) {
  const T* p = (const T*)base + at;
  if (vec && left >= 4) {
    unpack_vec<T, 4>(*(const VecOf<T, 4>*)p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? to_f(p[i]) : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void sel_store4(void* base, long long at, bool vec, int left, const float* v) {
  T* p = (T*)base + at;
  if (vec && left >= 4) {
    *(VecOf<T, 4>*)p = pack_vec<T, 4>(v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = from_f<T>(v[i]);
  }
}
__device__ __forceinline__ float4 f4(const float* v) { return make_float4(v[0], v[1], v[2], v[3]); }

// Where a thread stands: grid (chunk, b, group, tile), tile fastest.
template <class T, int L>
struct SelThread {
  static constexpr int SP = 4 * L;             // padded states
  static constexpr int ROWS = L;               // rows that a block stages at once (threads / (CH / 4))
  static constexpr int NI = ROWS >= kSelSeg ? 1 : kSelSeg / ROWS;
  const SelArgs& p;
  int tid, lane, warp, sg, cl;                 // state group, first of the thread's channels in the tile
  int tile, g, b, chunk, n0, nn;               // first channel of the tile, channels of the tile there are
  int t0, t1, len;                             // the chunk's rows; rows of the sequence
  int col, row, left;                          // staging: columns 4 col .. of rows row, row + ROWS, ..
  __device__ __forceinline__ SelThread(const SelArgs& p_) : p(p_) {
    tid = threadIdx.x;
    lane = tid & 31;
    warp = tid >> 5;
    sg = lane % L;
    cl = (warp * (32 / L) + lane / L) * 4;
    long long i = blockIdx.x;
    tile = (int)(i % p.tiles);
    i /= p.tiles;
    g = (int)(i % p.G);
    i /= p.G;
    b = (int)(i % p.B);
    chunk = (int)(i / p.B);
    n0 = g * p.Dg + tile * p.CH;
    nn = min(p.CH, p.Dg - tile * p.CH);
    t0 = chunk * p.steps;
    t1 = min(p.T, t0 + p.steps);
    len = row_length(p.lengths, p.wide, b, p.T);
    const int cv = p.CH / 4;
    col = tid % cv;
    row = tid / cv;
    left = max(0, min(4, nn - 4 * col));
  }
  // element (channel c, state s) of the thread: is it there, and where in (.., N, S)
  __device__ __forceinline__ bool there(int c, int s) const { return cl + c < nn && 4 * sg + s < p.S; }
  __device__ __forceinline__ size_t at(int c, int s) const { return (size_t)(n0 + cl + c) * p.S + 4 * sg + s; }
  __device__ __forceinline__ void load_state(const float* base, size_t lead, float (*h)[4]) const {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int s = 0; s < 4; ++s) h[c][s] = base && there(c, s) ? base[lead * p.N * p.S + at(c, s)] : 0.f;
  }
  __device__ __forceinline__ void store_state(float* base, size_t lead, const float (*h)[4]) const {
    const bool four = p.S % 4 == 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (four) {
        if (there(c, 0)) *(float4*)(base + lead * p.N * p.S + at(c, 0)) = f4(h[c]);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
          if (there(c, s)) base[lead * p.N * p.S + at(c, s)] = h[c][s];
      }
    }
  }
  __device__ __forceinline__ void load_decay(float (*A2)[4]) const {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int s = 0; s < 4; ++s) A2[c][s] = there(c, s) ? p.A[at(c, s)] * kLog2e : 0.f;
  }
  // rows of B or C of a segment, 0 past the sequence's end and past S
  __device__ __forceinline__ void stage_bc(const void* base, long long st, long long sb, int seg, float* dst) const {
    for (int e = tid; e < kSelSeg * SP; e += blockDim.x) {
      const int t = seg + e / SP, s = e % SP;
      dst[e] = t < len && s < p.S ? to_f(((const T*)base)[t * st + b * sb + (long long)g * p.S + s]) : 0.f;
    }
  }
  __device__ __forceinline__ void load_bias(float* v) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p.bias && i < left ? p.bias[n0 + 4 * col + i] : 0.f;
  }
  // a segment's dt: delta (0 past the end, which leaves a state as it is) and its derivative
  __device__ __forceinline__ void delta4(const float* z, const float* bias, bool on, float* d, float* sig) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d[i] = sig[i] = 0.f;
      if (on && i < left) d[i] = sel_delta(z[i] + bias[i], p.softplus, sig[i]);
    }
  }
};

__host__ __device__ constexpr int sel_fwd_smem(int L, int CH) { return (3 * kSelSeg * CH + 2 * kSelSeg * 4 * L) * 4; }

// LOCAL: the chunk's map only (from a zero state), without C, the gate and y
template <class T, int L, bool LOCAL>
__global__ void __launch_bounds__(128) k_sel_fwd(const SelArgs p) {
  using Th = SelThread<T, L>;
  constexpr int SP = Th::SP, ROWS = Th::ROWS, NI = Th::NI;
  extern __shared__ float4 sm4[];
  __shared__ uint8_t s_cut[kSelSeg];
  Th th(p);
  const int CH = p.CH;
  float* s_d = (float*)sm4;
  float* s_x = s_d + kSelSeg * CH;
  float* s_g = s_x + kSelSeg * CH;
  float* s_B = s_g + kSelSeg * CH;
  float* s_C = s_B + kSelSeg * SP;
  const int end = min(th.t1, th.len), n = th.n0 + 4 * th.col;
  const size_t BN = (size_t)p.chunks * p.B;
  float A2[4][4], h[4][4], bias[4], Dv[4], sumd[4] = {};
  bool any_cut = false;
  th.load_decay(A2);
  th.load_bias(bias);
#pragma unroll
  for (int i = 0; i < 4; ++i) Dv[i] = p.D && th.cl + i < th.nn ? p.D[th.n0 + th.cl + i] : 0.f;
  if (LOCAL) th.load_state(nullptr, 0, h);
  else if (p.chunks > 1) th.load_state(p.loc, (size_t)th.chunk * p.B + th.b, h);
  else th.load_state(p.h0, th.b, h);

  for (int seg = th.t0; seg < end; seg += kSelSeg) {
    float x[NI][4], z[NI][4], u[NI][4];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = th.row + i * ROWS, t = seg + r;
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i][k] = z[i][k] = u[i][k] = 0.f;
      if (r < kSelSeg && t < end) {
        sel_load4<T>(p.x, t * p.x_t + th.b * p.x_b + n, p.vec, th.left, x[i]);
        sel_load4<T>(p.dt, t * p.dt_t + th.b * p.dt_b + n, p.vec, th.left, z[i]);
        if (!LOCAL && p.gate) sel_load4<T>(p.gate, t * p.u_t + th.b * p.u_b + n, p.vec, th.left, u[i]);
      }
    }
    th.stage_bc(p.Bm, p.bm_t, p.bm_b, seg, s_B);
    if (!LOCAL) th.stage_bc(p.Cm, p.cm_t, p.cm_b, seg, s_C);
    if (th.tid < kSelSeg)
      s_cut[th.tid] = p.resets && seg + th.tid < end ? p.resets[(size_t)(seg + th.tid) * p.B + th.b] : 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = th.row + i * ROWS;
      if (r < kSelSeg) {
        float d[4], sig[4];
        th.delta4(z[i], bias, seg + r < end, d, sig);
        *(float4*)(s_d + r * CH + 4 * th.col) = f4(d);
        *(float4*)(s_x + r * CH + 4 * th.col) = f4(x[i]);
        if (!LOCAL) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float sg, so;
            sigmoid_pair<Accurate<T>::value>(u[i][k], sg, so);
            u[i][k] = p.gate ? u[i][k] * sg : 1.f;
          }
          *(float4*)(s_g + r * CH + 4 * th.col) = f4(u[i]);
        }
      }
    }
    __syncthreads();
    if (!LOCAL && p.states) th.store_state(p.states, (size_t)(seg / kSelSeg) * p.B + th.b, h);
#pragma unroll 2
    for (int r = 0; r < kSelSeg; ++r) {
      if (s_cut[r]) {
        any_cut = true;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int s = 0; s < 4; ++s) h[c][s] = 0.f;
      }
      const float4 d4 = *(const float4*)(s_d + r * CH + th.cl), x4 = *(const float4*)(s_x + r * CH + th.cl);
      const float4 B4 = *(const float4*)(s_B + r * SP + 4 * th.sg);
      const float d[4] = {d4.x, d4.y, d4.z, d4.w}, dx[4] = {d4.x * x4.x, d4.y * x4.y, d4.z * x4.z, d4.w * x4.w};
      const float Bv[4] = {B4.x, B4.y, B4.z, B4.w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int s = 0; s < 4; ++s) h[c][s] = fmaf(sel_exp2(d[c] * A2[c][s]), h[c][s], dx[c] * Bv[s]);
      if (LOCAL) {
#pragma unroll
        for (int c = 0; c < 4; ++c) sumd[c] += d[c];
      } else {
        const float4 C4 = *(const float4*)(s_C + r * SP + 4 * th.sg);
        const float Cv[4] = {C4.x, C4.y, C4.z, C4.w};
        float o[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          o[c] = Cv[0] * h[c][0];
#pragma unroll
          for (int s = 1; s < 4; ++s) o[c] = fmaf(Cv[s], h[c][s], o[c]);
          if (th.sg == 0) o[c] = fmaf(Dv[c], c == 0 ? x4.x : c == 1 ? x4.y : c == 2 ? x4.z : x4.w, o[c]);
        }
        sel_sum<1, L, 4>(o, th.lane);
        if (sel_first<1, L, 4>(th.lane)) {
          constexpr int NV = L >= 4 ? 1 : 4 / L;
          float* q = s_g + r * CH + th.cl + sel_owner<1, L, 4>(th.lane);
#pragma unroll
          for (int i = 0; i < NV; ++i) q[i] *= o[i];
        }
      }
    }
    __syncthreads();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = th.row + i * ROWS, t = seg + r;
        if (r < kSelSeg && t < end) {
          const float4 v = *(const float4*)(s_g + r * CH + 4 * th.col);
          const float o[4] = {v.x, v.y, v.z, v.w};
          sel_store4<T>(p.y, t * p.y_t + th.b * p.y_b + n, p.vec, th.left, o);
        }
      }
      __syncthreads();
    }
  }
  if (LOCAL) {
    const size_t lead = (size_t)th.chunk * p.B + th.b;
    th.store_state(p.loc, lead, h);
    if (th.sg == 0)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (th.cl + c < th.nn) p.sumd[lead * p.N + th.n0 + th.cl + c] = sumd[c];
    if (th.tid == 0 && th.tile == 0 && th.g == 0) p.cut[lead] = any_cut;
    return;
  }
  const float zero[4] = {};
  for (int t = max(th.t0, end) + th.row; t < th.t1; t += ROWS)
    sel_store4<T>(p.y, t * p.y_t + th.b * p.y_b + n, p.vec, th.left, zero);
  if (th.chunk == max(th.len - 1, 0) / p.steps) th.store_state(p.hT, th.b, h);
}

// The states (BACK: the gradients of the states) in front of (behind) each chunk, in place of its
// own share: one thread per (b, n, s), in time order.  start: h0 or ghT.
template <bool BACK>
__global__ void __launch_bounds__(256) k_sel_join(const SelArgs p, const float* __restrict__ start) {
  const size_t row = (size_t)p.N * p.S, all = row * p.B;
  const size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  if (i >= all) return;
  const int b = (int)(i / row);
  const size_t ns = i % row, n = ns / p.S;
  const float A2 = p.A[ns] * kLog2e;
  float h = start ? start[i] : 0.f;
  constexpr int U = 8;
  for (int c0 = 0; c0 < p.chunks; c0 += U) {
    float loc[U], a[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int c = BACK ? p.chunks - 1 - (c0 + k) : c0 + k;
      loc[k] = a[k] = 0.f;
      if (c0 + k < p.chunks) {
        const size_t lead = (size_t)c * p.B + b;
        loc[k] = p.loc[lead * row + ns];
        a[k] = p.cut[lead] ? -1.f : sel_exp2(A2 * p.sumd[lead * p.N + n]);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int c = BACK ? p.chunks - 1 - (c0 + k) : c0 + k;
      if (c0 + k < p.chunks) {
        p.loc[((size_t)c * p.B + b) * row + ns] = h;
        h = a[k] < 0.f ? loc[k] : fmaf(a[k], h, loc[k]);
      }
    }
  }
}

__host__ __device__ constexpr int sel_bwd_smem(int L, int CH, int warps, bool local) {
  return ((local ? 2 : 5) * kSelSeg * CH + 2 * kSelSeg * 4 * L) * 4 +
         (local ? 0 : (warps * kSelSeg * 2 * 4 * L) * 4 + kSelSeg * 4 * warps * 32 * 16);
}

// LOCAL: the chunk's share of the states' gradients only (from a zero gradient behind it)
template <class T, int L, bool LOCAL>
__global__ void __launch_bounds__(64) k_sel_bwd(const SelArgs p) {
  using Th = SelThread<T, L>;
  constexpr int SP = Th::SP, ROWS = Th::ROWS, NI = Th::NI, CG = 32 / L;
  extern __shared__ float4 sm4[];
  __shared__ uint8_t s_cut[kSelSeg];
  Th th(p);
  const int CH = p.CH, nt = blockDim.x, W = nt / 32;
  float4* hist = sm4;                                            // [kSelSeg][4][nt]: the state before each step
  float* s_d = (float*)(LOCAL ? sm4 : sm4 + kSelSeg * 4 * nt);
  float* s_go = s_d + kSelSeg * CH;                              // gy silu(gate); LOCAL: the last array
  float* s_C = s_go + kSelSeg * CH;
  float* s_B = s_C + kSelSeg * SP;
  float* s_x = s_B + kSelSeg * SP;
  float* s_ds = s_x + kSelSeg * CH;                              // gy silu'(gate)
  float* s_sg = s_ds + kSelSeg * CH;                             // d delta / d dt
  float* s_red = s_sg + kSelSeg * CH;                            // [W][kSelSeg][2 SP]
  const int end = min(th.t1, th.len), n = th.n0 + 4 * th.col;
  const size_t lead = (size_t)th.chunk * p.B + th.b;
  float A2[4][4], G[4][4], dA[4][4] = {}, bias[4], sumd[4] = {};
  constexpr int NV = L >= 4 ? 1 : 4 / L;
  const int own = sel_owner<1, L, 4>(th.lane);
  const bool first = sel_first<1, L, 4>(th.lane);
  float Do[NV], dDo[NV] = {}, dbo[NV] = {};
  bool any_cut = false;
  th.load_decay(A2);
  th.load_bias(bias);
#pragma unroll
  for (int i = 0; i < NV; ++i) Do[i] = p.D && th.cl + own + i < th.nn ? p.D[th.n0 + th.cl + own + i] : 0.f;
  if (LOCAL) th.load_state(nullptr, 0, G);
  else if (p.chunks > 1) th.load_state(p.loc, lead, G);
  else th.load_state(p.ghT, th.b, G);

  if (!LOCAL) {   // rows past the end: zero gradients
    const float zero[4] = {};
    for (int t = max(th.t0, end) + th.row; t < th.t1; t += ROWS) {
      if (p.dx) sel_store4<T>(p.dx, t * p.dx_t + th.b * p.dx_b + n, p.vec, th.left, zero);
      if (p.ddt) sel_store4<T>(p.ddt, t * p.ddt_t + th.b * p.ddt_b + n, p.vec, th.left, zero);
      if (p.dgate) sel_store4<T>(p.dgate, t * p.du_t + th.b * p.du_b + n, p.vec, th.left, zero);
    }
  }
  // dB and dC of all rows of the chunk are written, zeros past the end
  const auto write_bc = [&](int seg, int rows) {
    for (int e = th.tid; e < rows * 2 * SP; e += nt) {
      const int r = e / (2 * SP), q = e % (2 * SP), s = q % SP, t = seg + r;
      if (s < p.S) {
        float v = 0.f;
        if (t < end)
          for (int w = 0; w < W; ++w) v += s_red[(w * kSelSeg + r) * 2 * SP + q];
        float* dst = q < SP ? p.dB : p.dC;
        if (dst) dst[((((size_t)th.tile * p.T + t) * p.B + th.b) * p.G + th.g) * p.S + s] = v;
      }
    }
  };
  const int segs = end > th.t0 ? (end - th.t0 + kSelSeg - 1) / kSelSeg : 0;
  if (!LOCAL && (p.dB || p.dC))
    for (int seg = th.t0 + segs * kSelSeg; seg < th.t1; seg += kSelSeg) write_bc(seg, min(kSelSeg, th.t1 - seg));

  for (int k = segs - 1; k >= 0; --k) {
    const int seg = th.t0 + k * kSelSeg;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = th.row + i * ROWS, t = seg + r;
      if (r < kSelSeg) {
        float x[4] = {}, z[4] = {}, u[4] = {}, g[4] = {}, d[4], sig[4], gs[4];
        const bool on = t < end;
        if (on) {
          if (!LOCAL) sel_load4<T>(p.x, t * p.x_t + th.b * p.x_b + n, p.vec, th.left, x);
          sel_load4<T>(p.dt, t * p.dt_t + th.b * p.dt_b + n, p.vec, th.left, z);
          if (p.gate) sel_load4<T>(p.gate, t * p.u_t + th.b * p.u_b + n, p.vec, th.left, u);
          if (p.gy) sel_load4<T>(p.gy, t * p.gy_t + th.b * p.gy_b + n, p.vec, th.left, g);
        }
        th.delta4(z, bias, on, d, sig);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float sg, so;
          sigmoid_pair<Accurate<T>::value>(u[q], sg, so);
          gs[q] = g[q] * (sg * (1.f + u[q] * so));
          g[q] *= p.gate ? u[q] * sg : 1.f;
        }
        const int o = r * CH + 4 * th.col;
        *(float4*)(s_d + o) = f4(d);
        *(float4*)(s_go + o) = f4(g);
        if (!LOCAL) {
          *(float4*)(s_x + o) = f4(x);
          *(float4*)(s_ds + o) = f4(gs);
          *(float4*)(s_sg + o) = f4(sig);
        }
      }
    }
    th.stage_bc(p.Cm, p.cm_t, p.cm_b, seg, s_C);
    if (!LOCAL) th.stage_bc(p.Bm, p.bm_t, p.bm_b, seg, s_B);
    if (th.tid < kSelSeg)
      s_cut[th.tid] = p.resets && seg + th.tid < end ? p.resets[(size_t)(seg + th.tid) * p.B + th.b] : 0;
    float h[4][4];
    if (!LOCAL) th.load_state(p.states, (size_t)(seg / kSelSeg) * p.B + th.b, h);
    __syncthreads();
    if (!LOCAL) {
#pragma unroll 2
      for (int r = 0; r < kSelSeg; ++r) {
#pragma unroll
        for (int c = 0; c < 4; ++c) hist[(r * 4 + c) * nt + th.tid] = f4(h[c]);
        if (s_cut[r]) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int s = 0; s < 4; ++s) h[c][s] = 0.f;
        }
        const float4 d4 = *(const float4*)(s_d + r * CH + th.cl), x4 = *(const float4*)(s_x + r * CH + th.cl);
        const float4 B4 = *(const float4*)(s_B + r * SP + 4 * th.sg);
        const float d[4] = {d4.x, d4.y, d4.z, d4.w}, dx[4] = {d4.x * x4.x, d4.y * x4.y, d4.z * x4.z, d4.w * x4.w};
        const float Bv[4] = {B4.x, B4.y, B4.z, B4.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int s = 0; s < 4; ++s) h[c][s] = fmaf(sel_exp2(d[c] * A2[c][s]), h[c][s], dx[c] * Bv[s]);
        }
      }
    }
#pragma unroll 1
    for (int r = kSelSeg - 1; r >= 0; --r) {
      const float4 d4 = *(const float4*)(s_d + r * CH + th.cl), g4 = *(const float4*)(s_go + r * CH + th.cl);
      const float4 C4 = *(const float4*)(s_C + r * SP + 4 * th.sg);
      const float d[4] = {d4.x, d4.y, d4.z, d4.w}, go[4] = {g4.x, g4.y, g4.z, g4.w};
      const float Cv[4] = {C4.x, C4.y, C4.z, C4.w};
      const bool cut = s_cut[r];
      if (LOCAL) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          sumd[c] += d[c];
#pragma unroll
          for (int s = 0; s < 4; ++s)
            G[c][s] = cut ? 0.f : sel_exp2(d[c] * A2[c][s]) * fmaf(Cv[s], go[c], G[c][s]);
        }
        any_cut |= cut;
        continue;
      }
      const float4 x4 = *(const float4*)(s_x + r * CH + th.cl);
      const float4 B4 = *(const float4*)(s_B + r * SP + 4 * th.sg);
      const float dx[4] = {d4.x * x4.x, d4.y * x4.y, d4.z * x4.z, d4.w * x4.w}, Bv[4] = {B4.x, B4.y, B4.z, B4.w};
      float bc[8] = {}, gb[4], wa[4], o[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 q = hist[(r * 4 + c) * nt + th.tid];
        const float pre[4] = {q.x, q.y, q.z, q.w};
        gb[c] = wa[c] = o[c] = 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float a = sel_exp2(d[c] * A2[c][s]);
          const float Gt = fmaf(Cv[s], go[c], G[c][s]);
          o[c] = fmaf(Cv[s], h[c][s], o[c]);
          bc[4 + s] = fmaf(go[c], h[c][s], bc[4 + s]);
          bc[s] = fmaf(Gt, dx[c], bc[s]);
          gb[c] = fmaf(Gt, Bv[s], gb[c]);
          // nothing passes a reset, an infinite state neither
          const float ag = cut ? 0.f : a * Gt, w = cut ? 0.f : ag * pre[s];
          wa[c] = fmaf(w, A2[c][s], wa[c]);
          dA[c][s] = fmaf(w, d[c], dA[c][s]);
          G[c][s] = ag;
          h[c][s] = pre[s];
        }
      }
      sel_sum<L, 32, 8>(bc, th.lane);
      if (sel_first<L, 32, 8>(th.lane)) {
        constexpr int NB = CG >= 8 ? 1 : 8 / CG;
        const int j = sel_owner<L, 32, 8>(th.lane);   // values 0..3 are dB, 4..7 dC
#pragma unroll
        for (int i = 0; i < NB; ++i)
          s_red[(th.warp * kSelSeg + r) * 2 * SP + ((j + i) & 4 ? SP : 0) + 4 * th.sg + ((j + i) & 3)] = bc[i];
      }
      sel_sum<1, L, 4>(gb, th.lane);
      sel_sum<1, L, 4>(wa, th.lane);
      sel_sum<1, L, 4>(o, th.lane);
      __syncwarp();
      if (first) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = r * CH + th.cl + own + i;
          const float xx = s_x[e], gg = s_go[e];
          const float ddt = fmaf(gb[i], xx, wa[i] * kLn2) * s_sg[e];
          s_x[e] = fmaf(gb[i], s_d[e], Do[i] * gg);
          s_d[e] = ddt;
          s_ds[e] *= fmaf(Do[i], xx, o[i]);
          dDo[i] = fmaf(gg, xx, dDo[i]);
          dbo[i] += ddt;
        }
      }
    }
    __syncthreads();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = th.row + i * ROWS, t = seg + r;
        if (r < kSelSeg && t < end) {
          const int e = r * CH + 4 * th.col;
          if (p.dx) sel_store4<T>(p.dx, t * p.dx_t + th.b * p.dx_b + n, p.vec, th.left, s_x + e);
          if (p.ddt) sel_store4<T>(p.ddt, t * p.ddt_t + th.b * p.ddt_b + n, p.vec, th.left, s_d + e);
          if (p.dgate) sel_store4<T>(p.dgate, t * p.du_t + th.b * p.du_b + n, p.vec, th.left, s_ds + e);
        }
      }
      if (p.dB || p.dC) write_bc(seg, min(kSelSeg, th.t1 - seg));
      __syncthreads();
    }
  }
  if (LOCAL) {
    th.store_state(p.loc, lead, G);
    if (th.sg == 0)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (th.cl + c < th.nn) p.sumd[lead * p.N + th.n0 + th.cl + c] = sumd[c];
    if (th.tid == 0 && th.tile == 0 && th.g == 0) p.cut[lead] = any_cut;
    return;
  }
  if (p.dh0 && th.chunk == 0) th.store_state(p.dh0, th.b, G);
  if (p.dA) th.store_state(p.dA, lead, dA);
  if (first) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (th.cl + own + i < th.nn) {
        const size_t e = lead * p.N + th.n0 + th.cl + own + i;
        if (p.dD) p.dD[e] = dDo[i];
        if (p.db) p.db[e] = dbo[i];
      }
  }
}

// out[j] = sum over parts of part[k][j], in order.  Block: 32 columns by 32 runs of parts.
static __global__ void __launch_bounds__(1024) k_sel_sum(long long cols, long long parts, const float* __restrict__ part,
                                                  float* __restrict__ out) {
  __shared__ float sum[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const long long j = blockIdx.x * 32LL + lane;
  const long long p0 = parts * run / 32, p1 = parts * (run + 1) / 32;
  float s = 0.f;
  if (j < cols)
    for (long long q = p0; q < p1; ++q) s += part[q * cols + j];
  sum[run][lane] = s;
  __syncthreads();
  if (run == 0 && j < cols) {
    float t = 0.f;
    for (int r = 0; r < 32; ++r) t += sum[r][lane];
    out[j] = t;
  }
}
// dB and dC (T,B,G,S) from their partial sums, one to a tile of channels
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

// One time step: L lanes to a channel, four states a lane.  state and next (B,N,S) may be one tensor.
struct SelStep {
  int B, N, S, G, softplus, four;   // four: states in 16-byte accesses
  const void *x, *dt, *Bm, *Cm, *gate;
  const float *A, *D, *bias;
  const float* state;
  const uint8_t* active;
  void* y;
  float* next;
  long long x_b, dt_b, u_b, bm_b, cm_b;
};
template <class T, int L>
__global__ void __launch_bounds__(256) k_sel_step(const SelStep p) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  const long long ch = i / L;
  const int sg = (int)(i % L);
  const bool on = ch < (long long)p.B * p.N;
  const int b = on ? (int)(ch / p.N) : 0, n = on ? (int)(ch % p.N) : 0, g = n / (p.N / p.G);
  const bool act = on && (!p.active || p.active[b]);
  const long long at = ch * p.S + 4 * sg;
  float o = 0.f, x = 0.f;
  if (on) {
    float h[4] = {};
    const bool four = p.four;
    if (p.state) {
      if (four) {
        if (4 * sg < p.S) {
          const float4 v = *(const float4*)(p.state + at);
          h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
        }
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
          if (4 * sg + s < p.S) h[s] = p.state[at + s];
      }
    }
    if (act) {
      float sig;
      x = to_f(((const T*)p.x)[b * p.x_b + n]);
      const float d = sel_delta(to_f(((const T*)p.dt)[b * p.dt_b + n]) + (p.bias ? p.bias[n] : 0.f), p.softplus, sig);
      const T* Bp = (const T*)p.Bm + b * p.bm_b + (long long)g * p.S + 4 * sg;
      const T* Cp = (const T*)p.Cm + b * p.cm_b + (long long)g * p.S + 4 * sg;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (4 * sg + s < p.S) {
          h[s] = fmaf(sel_exp2(d * (p.A[(size_t)n * p.S + 4 * sg + s] * kLog2e)), h[s], d * x * to_f(Bp[s]));
          o = fmaf(to_f(Cp[s]), h[s], o);
        }
    }
    if (four) {
      if (4 * sg < p.S) *(float4*)(p.next + at) = f4(h);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (4 * sg + s < p.S) p.next[at + s] = h[s];
    }
  }
#pragma unroll
  for (int k = 1; k < L; k *= 2) o += __shfl_xor_sync(0xffffffffu, o, k);
  if (on && sg == 0) {
    float y = 0.f;
    if (act) {
      y = fmaf(p.D ? p.D[n] : 0.f, x, o);
      if (p.gate) {
        float s, so;
        const float u = to_f(((const T*)p.gate)[b * p.u_b + n]);
        sigmoid_pair<Accurate<T>::value>(u, s, so);
        y *= u * s;
      }
    }
    ((T*)p.y)[ch] = from_f<T>(y);
  }
}

}  // namespace delrec
