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
// A block of threads holds one row in registers and walks the rows of its grid stride;
// each tensor is read and written once (5 elements forward, 8 backward per channel), so
// HBM bounds it.  Sums are fp32: within a row a shuffle tree and one exchange through
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
  long long x_t, x_b, y_t, y_b, u_t, u_b;
  const float *w, *scale, *nw;          // each may be NULL (ones)
  void *out, *n;                        // x' and n; n may be NULL (no next norm)
  long long o_t, o_b, n_t, n_b;
  float *ry, *rx;                       // (T,B) 1/rms
  // backward
  const void *gx, *gn;
  long long gx_t, gx_b, gn_t, gn_b;
  void *dx, *dy, *du;
  long long dx_t, dx_b, dy_t, dy_b, du_t, du_b;
  float* part;                          // (grid, 2, N): Q and dw_next partials
};

template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* o) {
  const VecOf<T, V> r = *(const VecOf<T, V>*)p;
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
  slot = slot == 2 ? 0 : slot + 1;
  return s;
}

template <class T>
__device__ __forceinline__ float gate_value(float u, int kind) {
  float sg, so;
  sigmoid_pair<Accurate<T>::value>(u, sg, so);
  return kind == GATE_SIGMOID ? sg : u * sg;
}

// E = V * IT elements per thread: chunk k of V starts at (k * threads + thread) * V
template <class T, int V, int IT, bool GATE>
__global__ void __launch_bounds__(kNormThreads) k_norm_fwd(NormArgs p) {
  __shared__ float red[3][32];
  constexpr int E = V * IT;
  const int nth = blockDim.x, tid = threadIdx.x;
  const float inv_n = 1.f / (float)p.N;
  int slot = 0;
  float ws[E], nw[E];   // scale * w, w_next
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int c = (k * nth + tid) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool on = c + j < p.N;
      const float w = on ? (p.w ? p.w[c + j] : 1.f) : 0.f;
      ws[k * V + j] = w * (on && p.scale ? p.scale[c + j] : 1.f);
      nw[k * V + j] = on ? (p.nw ? p.nw[c + j] : 1.f) : 0.f;
    }
  }
  const long long rows = (long long)p.T * p.B;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const int t = (int)(r / p.B), b = (int)(r - (long long)t * p.B);
    const bool live = t < row_length(p.lengths, p.wide, b, p.T);
    float x[E], y[E], u[E];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int c = (k * nth + tid) * V;
      if (live && c < p.N) {
        load_vec<T, V>((const T*)p.x + t * p.x_t + b * p.x_b + c, x + k * V);
        if (p.y) {
          load_vec<T, V>((const T*)p.y + t * p.y_t + b * p.y_b + c, y + k * V);
          if (GATE) load_vec<T, V>((const T*)p.u + t * p.u_t + b * p.u_b + c, u + k * V);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[k * V + j] = y[k * V + j] = u[k * V + j] = 0.f;
      }
    }
    if (p.y) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf(y[i], y[i], s);
      const float ry = rsqrtf(block_sum(s, red, slot) * inv_n + p.eps);
      if (p.ry && tid == 0) p.ry[r] = ry;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float g = GATE ? ws[i] * gate_value<T>(u[i], p.kind) : ws[i];
        x[i] = live ? fmaf(y[i] * ry, g, x[i]) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * nth + tid) * V;
        if (c < p.N) store_vec<T, V>((T*)p.out + t * p.o_t + b * p.o_b + c, x + k * V);
      }
    }
    if (p.n) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf(x[i], x[i], s);
      const float rx = rsqrtf(block_sum(s, red, slot) * inv_n + p.eps);   // eps > 0: finite on a zero row
      if (p.rx && tid == 0) p.rx[r] = rx;
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * nth + tid) * V;
        if (c < p.N) {
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = x[k * V + j] * rx * nw[k * V + j];
          store_vec<T, V>((T*)p.n + t * p.n_t + b * p.n_b + c, o);
        }
      }
    }
  }
}

template <class T, int V, int IT, bool GATE>
__global__ void __launch_bounds__(kNormThreads) k_norm_bwd(NormArgs p) {
  __shared__ float red[3][32];
  constexpr int E = V * IT;
  const int nth = blockDim.x, tid = threadIdx.x;
  const float inv_n = 1.f / (float)p.N;
  int slot = 0;
  float ws[E], nw[E], q[E], qn[E];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int c = (k * nth + tid) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool on = c + j < p.N;
      const float w = on ? (p.w ? p.w[c + j] : 1.f) : 0.f;
      ws[k * V + j] = w * (on && p.scale ? p.scale[c + j] : 1.f);
      nw[k * V + j] = on ? (p.nw ? p.nw[c + j] : 1.f) : 0.f;
      q[k * V + j] = qn[k * V + j] = 0.f;
    }
  }
  const long long rows = (long long)p.T * p.B;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const int t = (int)(r / p.B), b = (int)(r - (long long)t * p.B);
    const bool live = t < row_length(p.lengths, p.wide, b, p.T);
    float x[E], y[E], u[E], g[E], v[E];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int c = (k * nth + tid) * V;
      const bool on = live && c < p.N;
#pragma unroll
      for (int j = 0; j < V; ++j) x[k * V + j] = y[k * V + j] = u[k * V + j] = g[k * V + j] = v[k * V + j] = 0.f;
      if (on) {
        if (p.gn) load_vec<T, V>((const T*)p.x + t * p.x_t + b * p.x_b + c, x + k * V);
        if (p.y) load_vec<T, V>((const T*)p.y + t * p.y_t + b * p.y_b + c, y + k * V);
        if (GATE && p.y) load_vec<T, V>((const T*)p.u + t * p.u_t + b * p.u_b + c, u + k * V);
        if (p.gx) load_vec<T, V>((const T*)p.gx + t * p.gx_t + b * p.gx_b + c, g + k * V);
        if (p.gn) load_vec<T, V>((const T*)p.gn + t * p.gn_t + b * p.gn_b + c, v + k * V);
      }
    }
    float ry = 0.f;
    if (p.y) {
      ry = p.ry[r];
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] *= ry;   // yh
    }
    if (p.gn) {
      const float rx = p.rx[r];
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (p.y) x[i] = fmaf(y[i], GATE ? ws[i] * gate_value<T>(u[i], p.kind) : ws[i], x[i]);
        x[i] *= rx;                             // xh
        qn[i] = fmaf(v[i], x[i], qn[i]);
        v[i] *= nw[i];
        s = fmaf(v[i], x[i], s);
      }
      s = block_sum(s, red, slot) * inv_n;
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = fmaf(rx, fmaf(-x[i], s, v[i]), g[i]);
    }
    if (!live) {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = 0.f;
    }
    if (p.dx) {
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int c = (k * nth + tid) * V;
        if (c < p.N) store_vec<T, V>((T*)p.dx + t * p.dx_t + b * p.dx_b + c, g + k * V);
      }
    }
    if (!p.y) continue;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float a = 1.f, da = 0.f;
      if (GATE) {
        float sg, so;
        sigmoid_pair<Accurate<T>::value>(u[i], sg, so);
        a = p.kind == GATE_SIGMOID ? sg : u[i] * sg;
        da = p.kind == GATE_SIGMOID ? sg * so : sg * fmaf(u[i], so, 1.f);
      }
      const float gy = g[i] * y[i];
      q[i] = fmaf(gy, a, q[i]);
      u[i] = gy * ws[i] * da;                   // du
      v[i] = g[i] * ws[i] * a;
      s = fmaf(v[i], y[i], s);
    }
    s = block_sum(s, red, slot) * inv_n;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int c = (k * nth + tid) * V;
      if (c < p.N) {
        if (p.dy) {
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = live ? ry * fmaf(-y[k * V + j], s, v[k * V + j]) : 0.f;
          store_vec<T, V>((T*)p.dy + t * p.dy_t + b * p.dy_b + c, o);
        }
        if (GATE && p.du) store_vec<T, V>((T*)p.du + t * p.du_t + b * p.du_b + c, u + k * V);
      }
    }
  }
  if (p.part) {
    float* o = p.part + (size_t)blockIdx.x * 2 * p.N;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int c = (k * nth + tid) * V;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < p.N) {
          o[c + j] = q[k * V + j];
          o[p.N + c + j] = qn[k * V + j];
        }
    }
  }
}

// dw = scale Q, dscale = w Q, dw_next from the blocks' partials, in block order: 32
// channels x 8 runs of blocks per thread block.
__global__ void __launch_bounds__(256) k_norm_dw(int N, int blocks, const float* __restrict__ part,
                                                 const float* __restrict__ w, const float* __restrict__ scale,
                                                 float* __restrict__ dw, float* __restrict__ dscale,
                                                 float* __restrict__ dnw) {
  __shared__ float sm[8][2][32];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float q = 0.f, qn = 0.f;
  if (c < N) {
    const int per = (blocks + 7) / 8, lo = run * per, hi = min(blocks, lo + per);
#pragma unroll 8
    for (int k = lo; k < hi; ++k) {
      q += part[(size_t)k * 2 * N + c];
      qn += part[(size_t)k * 2 * N + N + c];
    }
  }
  sm[run][0][lane] = q;
  sm[run][1][lane] = qn;
  __syncthreads();
  if (run == 0 && c < N) {
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      q += sm[k][0][lane];
      qn += sm[k][1][lane];
    }
    if (dw) dw[c] = q * (scale ? scale[c] : 1.f);
    if (dscale) dscale[c] = q * (w ? w[c] : 1.f);
    if (dnw) dnw[c] = qn;
  }
}

}  // namespace delrec
