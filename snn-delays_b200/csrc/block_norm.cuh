// RMS norms around a block, with the block's gate, residual scale and residual sum:
//
//   yh = y / sqrt(mean y^2 + eps),   x' = x + scale * act(u) * (yh * w)
//   n  = x' / sqrt(mean x'^2 + eps) * w_next          (next norm, optional)
//   act: 1, sigmoid(u) or u sigmoid(u).   Without y: x' = x, n = its norm.
//
//   backward, with the kept 1/rms of y and of x' (ry, rx), xh = x' rx:
//   G  = gx + rx (gn w_next - xh mean(gn w_next xh)),       dx = G
//   dy = ry (v - yh mean(v yh)),  v = G scale act w;   du = G scale yh w act'(u)
//   Q  = sum_rows G act yh:  dw = scale Q,  dscale = w Q;   dw_next = sum_rows gn xh
//
// A block of threads holds one row in registers, a vector of up to 16 bytes of each tensor per
// thread, and walks the rows of its grid stride, the next row on its way into shared
// memory meanwhile; each tensor is read and written once (5 elements forward, 8 backward per
// channel), so HBM bounds it.  Sums are fp32: within a row a shuffle tree and one exchange through
// shared memory; over rows per thread, then one partial per block and channel, summed in
// block order by a second kernel (no atomics: the same bits every time).  n is formed from
// the unrounded x'.
#pragma once

#include "seq_common.cuh"

namespace delrec {

enum : int { GATE_NONE = 0, GATE_SIGMOID = 1, GATE_SILU = 2 };
static constexpr int kNormThreads = 512;

struct NormArgs {
  int T, B, N, wide, kind;              // kind: the gate's function, where there is one
  float eps;
  const void* lengths;
  const void *x, *y, *u;
  int x_t, x_b, y_t, y_b, u_t, u_b;     // element strides
  const float *w, *scale, *nw;          // each may be NULL (ones)
  void *out, *n;                        // x' and n; n may be NULL (no next norm)
  int o_t, o_b, n_t, n_b;
  float *ry, *rx;                       // (T,B) 1/rms
  // backward
  const void *gx, *gn;
  int gx_t, gx_b, gn_t, gn_b;
  void *dx, *dy, *du;
  int dx_t, dx_b, dy_t, dy_b, du_t, du_b;
  float* part;                          // (grid, 2, N): Q and dw_next partials
};

template <class T, int V>
__device__ __forceinline__ void unpack_vec(const VecOf<T, V>& r, float* o) {
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = to_f(r.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* o) {
  VecOf<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = from_f<T>(o[i]);
  *(VecOf<T, V>*)p = r;
}

// A row's place: row = t * B + b, stepped by the grid without a division.
struct NormRow {
  int r, t, b;
  __device__ __forceinline__ void init(int row, int B) { r = row; t = row / B; b = row - t * B; }
  __device__ __forceinline__ void next(int step, int step_t, int step_b, int B) {
    r += step;
    t += step_t;
    b += step_b;
    if (b >= B) { b -= B; ++t; }
  }
};
template <class T>
__device__ __forceinline__ T* row_of(void* p, const NormRow& r, int st, int sb) {
  return (T*)p + ((long long)r.t * st + (long long)r.b * sb);
}
template <class T>
__device__ __forceinline__ const T* row_of(const void* p, const NormRow& r, int st, int sb) {
  return (const T*)p + ((long long)r.t * st + (long long)r.b * sb);
}

// The inputs of a row, NT tensors of IT vectors per thread.  Vectors of 4 bytes and more are
// copied into shared memory (cp.async) while the row before is worked on; every thread
// copies what it will read itself, so no barrier is needed.  One slot per tensor, vector and
// thread, two rows.
template <class T, int V, int IT, int NT>
struct NormStage {
  static constexpr int VB = V * (int)sizeof(T);
  static constexpr bool STAGED = VB >= 4 && IT <= 2;
  static constexpr int ROW = STAGED ? NT * IT * VB : 0;   // bytes per thread and row
  unsigned base;
  char* mem;
  __device__ __forceinline__ NormStage(char* m) : mem(m) {
    base = STAGED ? (unsigned)__cvta_generic_to_shared(m) : 0;
  }
  __device__ __forceinline__ int slot(int half, int ten, int k) const {
    return ((half * NT + ten) * IT + k) * (int)blockDim.x * VB + (int)threadIdx.x * VB;
  }
  __device__ __forceinline__ void copy(int half, int ten, const T* row, int N) const {
    if constexpr (STAGED) {
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * (int)blockDim.x + (int)threadIdx.x) * V;
        if (c < N) {
          if constexpr (VB == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + slot(half, ten, k)), "l"(row + c));
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(base + slot(half, ten, k)), "l"(row + c),
                         "n"(VB));
        }
      }
    }
  }
  __device__ __forceinline__ void commit() const {
    if (STAGED) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  template <int LEFT>
  __device__ __forceinline__ void wait() const {
    if (STAGED) asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
  }
  // vector k of tensor ten as floats; zeros past the row's end
  __device__ __forceinline__ void read(int half, int ten, int k, const T* row, int N, float* o) const {
    const int c = (k * (int)blockDim.x + (int)threadIdx.x) * V;
    if (c < N) {
      if constexpr (STAGED) unpack_vec<T, V>(*(const VecOf<T, V>*)(mem + slot(half, ten, k)), o);
      else unpack_vec<T, V>(*(const VecOf<T, V>*)(row + c), o);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = 0.f;
    }
  }
};

// Sum over the block, the same bits in every thread.  slot alternates between calls, so
// one barrier per sum is enough.
__device__ __forceinline__ float block_sum(float v, float (*red)[32], int& slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) red[slot][threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < nw; ++i) s += red[slot][i];
  slot ^= 1;
  return s;
}

// A gate's function and derivative from the folded sigmoid (its smaller side, signed as u).
struct GateVal {
  float a, da;
};
__device__ __forceinline__ GateVal gate_eval(float fold, float u, int kind) {
  float sg, so;
  gate_unfold(fold, sg, so);
  GateVal g;
  g.a = kind == GATE_SIGMOID ? sg : u * sg;
  g.da = kind == GATE_SIGMOID ? sg * so : sg * fmaf(u, so, 1.f);
  return g;
}

// E = V * IT elements per thread: vector k starts at channel (k * threads + thread) * V
template <class T, int V, int IT, bool GATE>
__global__ void __launch_bounds__(kNormThreads) k_norm_fwd(NormArgs p) {
  __shared__ float red[2][32];
  extern __shared__ __align__(16) char norm_stage[];
  constexpr int E = V * IT;
  using Stage = NormStage<T, V, IT, GATE ? 3 : 2>;
  const Stage st(norm_stage);
  const int nth = blockDim.x, tid = threadIdx.x, rows = p.T * p.B;
  const float inv_n = 1.f / (float)p.N;
  const int gs = gridDim.x, gt = gs / p.B, gb = gs - gt * p.B;
  int slot = 0;
  float ws[E], nw[E];   // scale * w, w_next
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (k * nth + tid) * V + j;
      const bool on = c < p.N;
      ws[k * V + j] = on ? (p.w ? p.w[c] : 1.f) * (p.scale ? p.scale[c] : 1.f) : 0.f;
      nw[k * V + j] = on ? (p.nw ? p.nw[c] : 1.f) : 0.f;
    }
  auto xr = [&](const NormRow& r) { return row_of<T>(p.x, r, p.x_t, p.x_b); };
  auto yr = [&](const NormRow& r) { return row_of<T>(p.y, r, p.y_t, p.y_b); };
  auto ur = [&](const NormRow& r) { return row_of<T>(p.u, r, p.u_t, p.u_b); };
  auto live_row = [&](const NormRow& r) { return !p.lengths || r.t < row_length(p.lengths, p.wide, r.b, p.T); };
  auto fetch = [&](const NormRow& r, int half, bool live) {
    if (live) {
      st.copy(half, 0, xr(r), p.N);
      if (p.y) st.copy(half, 1, yr(r), p.N);
      if (GATE && p.y) st.copy(half, 2, ur(r), p.N);
    }
    st.commit();
  };
  NormRow cur;
  cur.init(blockIdx.x, p.B);
  bool live = live_row(cur);
  fetch(cur, 0, live);
  for (int half = 0; cur.r < rows; half ^= 1) {
    NormRow nxt = cur;
    nxt.next(gs, gt, gb, p.B);
    const bool next_live = nxt.r < rows && live_row(nxt);
    fetch(nxt, half ^ 1, next_live);
    st.template wait<1>();
    float x[E], y[E], u[E];
    if (live) {
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        st.read(half, 0, k, xr(cur), p.N, x + k * V);
        if (p.y) st.read(half, 1, k, yr(cur), p.N, y + k * V);
        if (GATE && p.y) st.read(half, 2, k, ur(cur), p.N, u + k * V);
      }
      if (p.y) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(y[i], y[i], s);
        const float ry = rsqrtf(block_sum(s, red, slot) * inv_n + p.eps);
        if (p.ry && tid == 0) p.ry[cur.r] = ry;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float g = ws[i];
          if (GATE) {
            float sg, so;
            sigmoid_pair<Accurate<T>::value>(u[i], sg, so);
            g *= p.kind == GATE_SIGMOID ? sg : u[i] * sg;
          }
          x[i] = fmaf(y[i] * ry, g, x[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = 0.f;
    }
    if (p.y) {
      T* o = row_of<T>(p.out, cur, p.o_t, p.o_b);
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * nth + tid) * V;
        if (c < p.N) store_vec<T, V>(o + c, x + k * V);
      }
    }
    if (p.n) {
      float rx = 0.f;
      if (live) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(x[i], x[i], s);
        rx = rsqrtf(block_sum(s, red, slot) * inv_n + p.eps);
        if (p.rx && tid == 0) p.rx[cur.r] = rx;
      }
      T* o = row_of<T>(p.n, cur, p.n_t, p.n_b);
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * nth + tid) * V;
        if (c < p.N) {
          float v[V];
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = x[k * V + j] * rx * nw[k * V + j];
          store_vec<T, V>(o + c, v);
        }
      }
    }
    cur = nxt;
    live = next_live;
  }
  st.template wait<0>();
}

template <class T, int V, int IT, bool GATE>
__global__ void __launch_bounds__(kNormThreads) k_norm_bwd(NormArgs p) {
  __shared__ float red[2][32];
  extern __shared__ __align__(16) char norm_stage[];
  constexpr int E = V * IT;
  using Stage = NormStage<T, V, IT, GATE ? 5 : 4>;
  const Stage st(norm_stage);
  const int nth = blockDim.x, tid = threadIdx.x, rows = p.T * p.B;
  const float inv_n = 1.f / (float)p.N;
  const int gs = gridDim.x, gt = gs / p.B, gb = gs - gt * p.B;
  int slot = 0;
  float ws[E], nw[E], q[E], qn[E];
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (k * nth + tid) * V + j;
      const bool on = c < p.N;
      ws[k * V + j] = on ? (p.w ? p.w[c] : 1.f) * (p.scale ? p.scale[c] : 1.f) : 0.f;
      nw[k * V + j] = on ? (p.nw ? p.nw[c] : 1.f) : 0.f;
      q[k * V + j] = qn[k * V + j] = 0.f;
    }
  auto xr = [&](const NormRow& r) { return row_of<T>(p.x, r, p.x_t, p.x_b); };
  auto yr = [&](const NormRow& r) { return row_of<T>(p.y, r, p.y_t, p.y_b); };
  auto ur = [&](const NormRow& r) { return row_of<T>(p.u, r, p.u_t, p.u_b); };
  auto gxr = [&](const NormRow& r) { return row_of<T>(p.gx, r, p.gx_t, p.gx_b); };
  auto gnr = [&](const NormRow& r) { return row_of<T>(p.gn, r, p.gn_t, p.gn_b); };
  auto live_row = [&](const NormRow& r) { return !p.lengths || r.t < row_length(p.lengths, p.wide, r.b, p.T); };
  float ry_ahead = 0.f, rx_ahead = 0.f;
  auto fetch = [&](const NormRow& r, int half, bool live) {
    if (live) {
      if (p.gx) st.copy(half, 0, gxr(r), p.N);
      if (p.gn) {
        st.copy(half, 1, gnr(r), p.N);
        st.copy(half, 2, xr(r), p.N);
        rx_ahead = p.rx[r.r];
      }
      if (p.y) {
        st.copy(half, 3, yr(r), p.N);
        if (GATE) st.copy(half, 4, ur(r), p.N);
        ry_ahead = p.ry[r.r];
      }
    }
    st.commit();
  };
  NormRow cur;
  cur.init(blockIdx.x, p.B);
  bool live = live_row(cur);
  fetch(cur, 0, live);
  for (int half = 0; cur.r < rows; half ^= 1) {
    const float ry = ry_ahead, rx = rx_ahead;
    NormRow nxt = cur;
    nxt.next(gs, gt, gb, p.B);
    const bool next_live = nxt.r < rows && live_row(nxt);
    fetch(nxt, half ^ 1, next_live);
    T* dx = p.dx ? row_of<T>(p.dx, cur, p.dx_t, p.dx_b) : nullptr;
    T* dy = p.dy ? row_of<T>(p.dy, cur, p.dy_t, p.dy_b) : nullptr;
    T* du = GATE && p.du ? row_of<T>(p.du, cur, p.du_t, p.du_b) : nullptr;
    if (!live) {
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * nth + tid) * V;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.f;
        if (c < p.N) {
          if (dx) store_vec<T, V>(dx + c, o);
          if (dy) store_vec<T, V>(dy + c, o);
          if (du) store_vec<T, V>(du + c, o);
        }
      }
      cur = nxt;
      live = next_live;
      continue;
    }
    st.template wait<1>();
    float y[E], fold[E], g[E];
    if (p.y) {
#pragma unroll
      for (int k = 0; k < IT; ++k) st.read(half, 3, k, yr(cur), p.N, y + k * V);
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] *= ry;   // yh
      if (GATE) {
#pragma unroll
        for (int k = 0; k < IT; ++k) st.read(half, 4, k, ur(cur), p.N, fold + k * V);
#pragma unroll
        for (int i = 0; i < E; ++i) fold[i] = gate_fold<Accurate<T>::value>(fold[i]);
      }
    }
    // u is read again where it is needed beside its gate (silu)
    auto u_of = [&](int k, float* o) { st.read(half, 4, k, ur(cur), p.N, o); };
#pragma unroll
    for (int i = 0; i < E; ++i) g[i] = 0.f;
    if (p.gx) {
#pragma unroll
      for (int k = 0; k < IT; ++k) st.read(half, 0, k, gxr(cur), p.N, g + k * V);
    }
    if (p.gn) {
      float xh[E], v[E];
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        float u[V];
        st.read(half, 2, k, xr(cur), p.N, xh + k * V);
        st.read(half, 1, k, gnr(cur), p.N, v + k * V);
        if (GATE && p.y) u_of(k, u);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int i = k * V + j;
          if (p.y) xh[i] = fmaf(y[i], GATE ? ws[i] * gate_eval(fold[i], u[j], p.kind).a : ws[i], xh[i]);
          xh[i] *= rx;
          qn[i] = fmaf(v[i], xh[i], qn[i]);
          v[i] *= nw[i];
          s = fmaf(v[i], xh[i], s);
        }
      }
      s = block_sum(s, red, slot) * inv_n;
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = fmaf(rx, fmaf(-xh[i], s, v[i]), g[i]);
    }
    if (dx) {
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * nth + tid) * V;
        if (c < p.N) store_vec<T, V>(dx + c, g + k * V);
      }
    }
    if (p.y) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        float u[V], o[V];
        if (GATE) u_of(k, u);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int i = k * V + j;
          GateVal gv{1.f, 0.f};
          if (GATE) gv = gate_eval(fold[i], u[j], p.kind);
          const float gy = g[i] * y[i];
          q[i] = fmaf(gy, gv.a, q[i]);
          o[j] = gy * ws[i] * gv.da;            // du
          g[i] *= ws[i] * gv.a;                 // v
          s = fmaf(g[i], y[i], s);
        }
        const int c = (k * nth + tid) * V;
        if (GATE && du && c < p.N) store_vec<T, V>(du + c, o);
      }
      s = block_sum(s, red, slot) * inv_n;
      if (dy) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          const int c = (k * nth + tid) * V;
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = ry * fmaf(-y[k * V + j], s, g[k * V + j]);
          if (c < p.N) store_vec<T, V>(dy + c, o);
        }
      }
    }
    cur = nxt;
    live = next_live;
  }
  st.template wait<0>();
  if (p.part) {
    float* o = p.part + (size_t)blockIdx.x * 2 * p.N;
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (k * nth + tid) * V + j;
        if (c < p.N) {
          o[c] = q[k * V + j];
          o[p.N + c] = qn[k * V + j];
        }
      }
  }
}

// dw = scale Q, dscale = w Q (blockIdx.y = 0) and dw_next (1) from the blocks' partials: 32
// channels and 32 runs of blocks per thread block, summed in a fixed order.
__global__ void __launch_bounds__(1024) k_norm_dw(int N, int blocks, const float* __restrict__ part,
                                                  const float* __restrict__ w, const float* __restrict__ scale,
                                                  float* __restrict__ dw, float* __restrict__ dscale,
                                                  float* __restrict__ dnw) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < N) {
    const float* q = part + (size_t)blockIdx.y * N + c;
#pragma unroll 8
    for (int k = run; k < blocks; k += 32) s += q[(size_t)k * 2 * N];
  }
  sm[run][lane] = s;
  __syncthreads();
  s = sm[lane][run];   // channel run of this block, run lane
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int d = blockIdx.x * 32 + run;
  if (lane == 0 && d < N) {
    if (blockIdx.y) {
      if (dnw) dnw[d] = s;
    } else {
      if (dw) dw[d] = s * (scale ? scale[d] : 1.f);
      if (dscale) dscale[d] = s * (w ? w[d] : 1.f);
    }
  }
}

}  // namespace delrec
