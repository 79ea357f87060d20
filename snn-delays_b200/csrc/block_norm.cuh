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
// the unrounded x'.  Measured, forward / backward: T=250 B=256 N=512 fp32 115 / 165 us (5.7 / 6.3
// TB/s); T=784 B=64 N=2048 bf16 166 / 341 us (6.2 / 4.8 TB/s), the latter bound by issue slots at the
// 16 warps that 128 registers leave an SM.  A norm alone, 64000 x 512: fp32 45 / 98 us (5.8 / 4.0 TB/s),
// bf16 31 / 66 (4.2 / 3.0).
//
// Rows past 512 threads of 16 bytes hold 16 and 32 channels to a thread, more than the registers:
// the backward spills from 16 on, the forward at 32 (32 M elements, N = 4096 / 8192 / 16384:
// fp32 backward 172 / 294 / 978 us, bf16 at 64 M 244 / 328 / 1277; forward fp32 116 / 155 / 203, bf16
// 113 / 116 / 360).  16-bit rows of odd widths go an element at a time (fp16, 64000 rows: N = 700
// 104 / 164 us, N = 702 522 / 778).
#pragma once

#include <string.h>

#include "seq_common.cuh"

namespace delrec {

enum : int { GATE_NONE = 0, GATE_SIGMOID = 1, GATE_SILU = 2 };
static constexpr int kNormThreads = 512;

struct NormArgs {
  int T, B, N, wide, kind;              // kind: the gate's function, where there is one
  int pitch;                            // of rows, where all tensors share it (FLAT)
  int slots;                            // rows in shared memory: one at work, the others on their way
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
__device__ __forceinline__ void store_vec(T* p, const float* o) {
  *(VecOf<T, V>*)p = pack_vec<T, V>(o);
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
// This thread's first channel c0 of a row.  FLAT: every tensor's rows lie pitch apart, less
// than 2^31 elements in all, so one 32-bit offset serves them all.
template <class T, bool FLAT>
__device__ __forceinline__ T* row_of(const NormArgs& a, void* p, const NormRow& r, int st, int sb, int c0) {
  if (FLAT) return (T*)p + (r.r * a.pitch + c0);
  return (T*)p + ((long long)r.t * st + (long long)r.b * sb + c0);
}
template <class T, bool FLAT>
__device__ __forceinline__ const T* row_of(const NormArgs& a, const void* p, const NormRow& r, int st, int sb, int c0) {
  if (FLAT) return (const T*)p + (r.r * a.pitch + c0);
  return (const T*)p + ((long long)r.t * st + (long long)r.b * sb + c0);
}

// The inputs of a row, NT tensors of IT vectors per thread.  Vectors of 4 bytes and more are
// copied into shared memory (cp.async) while rows before are worked on; every thread
// copies what it will read itself, so no barrier is needed.  A vector of all threads lies side
// by side: copies that scatter a thread's vectors over shared memory cost a third more time.
template <class T, int V, int IT, int NT>
struct NormStage {
  static constexpr int VB = V * (int)sizeof(T);
  static constexpr bool STAGED = VB >= 4 && VB * IT <= 32;   // two rows of 5 tensors and 512 threads fit 160 KB
  static constexpr int ROW = STAGED ? NT * IT * VB : 0;   // bytes per thread and row
  unsigned base;
  const char* mem;
  int plane, size;   // bytes of one vector of all threads, of a slot
  __device__ __forceinline__ NormStage(char* m) {
    plane = blockDim.x * VB;
    size = blockDim.x * ROW;
    mem = m + threadIdx.x * VB;
    base = STAGED ? (unsigned)__cvta_generic_to_shared(mem) : 0;
  }
  // zeros, once, in the slots of vectors past the row's end: reads need no test
  __device__ __forceinline__ void clear(int slots, int left, int nthV) const {
    if constexpr (STAGED) {
#pragma unroll
      for (int k = 0; k < IT; ++k)
        if (k * nthV >= left)
          for (int i = 0; i < slots * NT; ++i)
            memset(const_cast<char*>(mem) + i / NT * size + (i % NT * IT + k) * plane, 0, VB);
    }
  }
  // col: this thread's first channel in the row
  __device__ __forceinline__ void copy(unsigned at, int ten, const T* col, int left, int nthV) const {
    if constexpr (STAGED) {
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        if (k * nthV < left) {
          if constexpr (VB == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + (ten * IT + k) * plane), "l"(col + k * nthV));
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at + (ten * IT + k) * plane),
                         "l"(col + k * nthV), "n"(VB));
        }
      }
    }
  }
  __device__ __forceinline__ void commit() const {
    if (STAGED) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // until the row at work is there: the slots - 1 rows copied after it may be on their way
  __device__ __forceinline__ void wait(int slots) const {
    if (!STAGED) return;
    if (slots == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (slots == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  // vector k of tensor ten as floats; zeros past the row's end
  __device__ __forceinline__ void read(const char* at, int ten, int k, const T* col, int left, int nthV, float* o) const {
    if constexpr (STAGED) {
      unpack_vec<T, V>(*(const VecOf<T, V>*)(at + (ten * IT + k) * plane), o);
    } else if (k * nthV < left) {
      unpack_vec<T, V>(*(const VecOf<T, V>*)(col + k * nthV), o);
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
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (nw == 1) return v;
  if (lane == 0) red[slot][threadIdx.x >> 5] = v;
  __syncthreads();
  v = (lane & 15) < nw ? red[slot][lane & 15] : 0.f;   // both halves of the warp
  slot ^= 1;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);   // at most 16 warps
  return v;
}

// Three sums at once.
__device__ __forceinline__ void block_sum3(float (&v)[3], float (*red)[32], int& slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (nw == 1) return;
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < 3; ++k) red[slot * 3 + k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = (lane & 15) < nw ? red[slot * 3 + k][lane & 15] : 0.f;
  slot ^= 1;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

// E = V * IT elements per thread: vector k starts at channel (k * threads + thread) * V.
// KIND: GATE_*.
template <class T, int V, int IT, int KIND, bool FLAT>
__global__ void __launch_bounds__(kNormThreads) k_norm_fwd(NormArgs p) {
  __shared__ float red[2][32];
  extern __shared__ __align__(16) char norm_stage[];
  constexpr int E = V * IT;
  constexpr bool GATE = KIND != GATE_NONE;
  using Stage = NormStage<T, V, IT, GATE ? 3 : 2>;
  const Stage st(norm_stage);
  const int nthV = blockDim.x * V, c0 = threadIdx.x * V, left = p.N - c0, rows = p.T * p.B;
  const float inv_n = 1.f / (float)p.N;
  const int gs = gridDim.x, gt = gs / p.B, gb = gs - gt * p.B;
  int slot = 0;
  float ws[E], nw[E];   // scale * w, w_next
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = c0 + k * nthV + j;
      const bool on = c < p.N;
      ws[k * V + j] = on ? (p.w ? p.w[c] : 1.f) * (p.scale ? p.scale[c] : 1.f) : 0.f;
      nw[k * V + j] = on ? (p.nw ? p.nw[c] : 1.f) : 0.f;
    }
  auto xr = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.x, r, p.x_t, p.x_b, c0); };
  auto yr = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.y, r, p.y_t, p.y_b, c0); };
  auto ur = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.u, r, p.u_t, p.u_b, c0); };
  auto live_row = [&](const NormRow& r) { return !p.lengths || r.t < row_length(p.lengths, p.wide, r.b, p.T); };
  auto fetch = [&](const NormRow& r, unsigned at, bool live) {
    if (live) {
      st.copy(at, 0, xr(r), left, nthV);
      if (p.y) {
        st.copy(at, 1, yr(r), left, nthV);
        if (GATE) st.copy(at, 2, ur(r), left, nthV);
      }
    }
    st.commit();
  };
  st.clear(p.slots, left, nthV);
  NormRow cur, ahead;
  cur.init(blockIdx.x, p.B);
  ahead = cur;
  unsigned lives = 0;   // bit k: row k of those under way, from the one at work on
  for (int k = 0; k < p.slots - 1; ++k) {
    const bool l = ahead.r < rows && live_row(ahead);
    lives |= (unsigned)l << k;
    fetch(ahead, st.base + k * st.size, l);
    ahead.next(gs, gt, gb, p.B);
  }
  for (int slot_now = 0; cur.r < rows; slot_now = slot_now == p.slots - 1 ? 0 : slot_now + 1) {
    const bool live = lives & 1;
    const bool l = ahead.r < rows && live_row(ahead);
    fetch(ahead, st.base + (slot_now ? slot_now - 1 : p.slots - 1) * st.size, l);
    lives = (lives >> 1) | (unsigned)l << (p.slots - 2);
    ahead.next(gs, gt, gb, p.B);
    const char* at = st.mem + slot_now * st.size;
    st.wait(p.slots);
    float x[E], y[E], u[E];
    if (live) {
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        st.read(at, 0, k, xr(cur), left, nthV, x + k * V);
        if (p.y) {
          st.read(at, 1, k, yr(cur), left, nthV, y + k * V);
          if (GATE) st.read(at, 2, k, ur(cur), left, nthV, u + k * V);
        }
      }
      if (p.y) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(y[i], y[i], s);
        const float ry = rsqrtf(block_sum(s, red, slot) * inv_n + p.eps);
        if (p.ry && threadIdx.x == 0) p.ry[cur.r] = ry;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float g = ws[i];
          if (GATE) {
            float sg, so;
            sigmoid_pair<Accurate<T>::value>(u[i], sg, so);
            g *= KIND == GATE_SIGMOID ? sg : u[i] * sg;
          }
          x[i] = fmaf(y[i] * ry, g, x[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = 0.f;
    }
    if (p.y) {
      T* o = row_of<T, FLAT>(p, p.out, cur, p.o_t, p.o_b, c0);
#pragma unroll
      for (int k = 0; k < IT; ++k)
        if (k * nthV < left) store_vec<T, V>(o + k * nthV, x + k * V);
    }
    if (p.n) {
      float rx = 0.f;
      if (live) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(x[i], x[i], s);
        rx = rsqrtf(block_sum(s, red, slot) * inv_n + p.eps);
        if (p.rx && threadIdx.x == 0) p.rx[cur.r] = rx;
      }
      T* o = row_of<T, FLAT>(p, p.n, cur, p.n_t, p.n_b, c0);
#pragma unroll
      for (int k = 0; k < IT; ++k)
        if (k * nthV < left) {
          float v[V];
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = x[k * V + j] * rx * nw[k * V + j];
          store_vec<T, V>(o + k * nthV, v);
        }
    }
    cur.next(gs, gt, gb, p.B);
  }
  st.wait(0);
}

// One barrier a row: with c = scale w act yh and g = gx + rx gn w_next, the sums that dx and
// dy need are S1 = sum gn w_next xh, S2 = sum g c and S3 = sum xh c, since G = g - rx (S1 / N) xh
// gives sum G c = S2 - rx (S1 / N) S3.  The difference loses no more than forming each G does
// (T=250 B=256 N=512 fp32, against float64, relative: dx 4.5e-8, dy 9.8e-8, du 1.0e-7, as much as two
// sweeps of fp32 operations; the weight gradients, sums of 64000 rows in fp32, 2.3e-7).
template <class T, int V, int IT, int KIND, bool FLAT>
__global__ void __launch_bounds__(kNormThreads) k_norm_bwd(NormArgs p) {
  __shared__ float red[6][32];
  extern __shared__ __align__(16) char norm_stage[];
  constexpr int E = V * IT;
  constexpr bool GATE = KIND != GATE_NONE;
  using Stage = NormStage<T, V, IT, GATE ? 5 : 4>;
  const Stage st(norm_stage);
  const int nthV = blockDim.x * V, c0 = threadIdx.x * V, left = p.N - c0, rows = p.T * p.B;
  const float inv_n = 1.f / (float)p.N;
  const int gs = gridDim.x, gt = gs / p.B, gb = gs - gt * p.B;
  int slot = 0;
  float ws[E], nw[E], q[E], qn[E];
#pragma unroll
  for (int k = 0; k < IT; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = c0 + k * nthV + j;
      const bool on = c < p.N;
      ws[k * V + j] = on ? (p.w ? p.w[c] : 1.f) * (p.scale ? p.scale[c] : 1.f) : 0.f;
      nw[k * V + j] = on ? (p.nw ? p.nw[c] : 1.f) : 0.f;
      q[k * V + j] = qn[k * V + j] = 0.f;
    }
  auto xr = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.x, r, p.x_t, p.x_b, c0); };
  auto yr = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.y, r, p.y_t, p.y_b, c0); };
  auto ur = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.u, r, p.u_t, p.u_b, c0); };
  auto gxr = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.gx, r, p.gx_t, p.gx_b, c0); };
  auto gnr = [&](const NormRow& r) { return row_of<T, FLAT>(p, p.gn, r, p.gn_t, p.gn_b, c0); };
  auto live_row = [&](const NormRow& r) { return !p.lengths || r.t < row_length(p.lengths, p.wide, r.b, p.T); };
  auto fetch = [&](const NormRow& r, unsigned at, bool live) {
    if (live) {
      if (p.gx) st.copy(at, 0, gxr(r), left, nthV);
      if (p.gn) {
        st.copy(at, 1, gnr(r), left, nthV);
        st.copy(at, 2, xr(r), left, nthV);
      }
      if (p.y) {
        st.copy(at, 3, yr(r), left, nthV);
        if (GATE) st.copy(at, 4, ur(r), left, nthV);
      }
    }
    st.commit();
  };
  st.clear(p.slots, left, nthV);
  NormRow cur, ahead;
  cur.init(blockIdx.x, p.B);
  ahead = cur;
  unsigned lives = 0;   // bit k: row k of those under way, from the one at work on
  for (int k = 0; k < p.slots - 1; ++k) {
    const bool l = ahead.r < rows && live_row(ahead);
    lives |= (unsigned)l << k;
    fetch(ahead, st.base + k * st.size, l);
    ahead.next(gs, gt, gb, p.B);
  }
  // the kept 1/rms of the row at work, read a row ahead
  auto kept = [&](int r, float& y, float& x) {
    if (r < rows) {
      if (p.y) y = p.ry[r];
      if (p.gn) x = p.rx[r];
    }
  };
  float ry_ahead = 0.f, rx_ahead = 0.f;
  kept(cur.r, ry_ahead, rx_ahead);
  for (int slot_now = 0; cur.r < rows; slot_now = slot_now == p.slots - 1 ? 0 : slot_now + 1) {
    const bool live = lives & 1;
    const float ry = ry_ahead, rx = rx_ahead;
    kept(cur.r + gs, ry_ahead, rx_ahead);
    const bool l = ahead.r < rows && live_row(ahead);
    fetch(ahead, st.base + (slot_now ? slot_now - 1 : p.slots - 1) * st.size, l);
    lives = (lives >> 1) | (unsigned)l << (p.slots - 2);
    ahead.next(gs, gt, gb, p.B);
    const char* at = st.mem + slot_now * st.size;
    T* dx = p.dx ? row_of<T, FLAT>(p, p.dx, cur, p.dx_t, p.dx_b, c0) : nullptr;
    T* dy = p.dy ? row_of<T, FLAT>(p, p.dy, cur, p.dy_t, p.dy_b, c0) : nullptr;
    T* du = GATE && p.du ? row_of<T, FLAT>(p, p.du, cur, p.du_t, p.du_b, c0) : nullptr;
    if (!live) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll
      for (int k = 0; k < IT; ++k)
        if (k * nthV < left) {
          if (dx) store_vec<T, V>(dx + k * nthV, o);
          if (dy) store_vec<T, V>(dy + k * nthV, o);
          if (du) store_vec<T, V>(du + k * nthV, o);
        }
      cur.next(gs, gt, gb, p.B);
      continue;
    }
    st.wait(p.slots);
    float y[E], a[E], da[E], g[E], xh[E];   // yh, act, act', the gradient, xh
    float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = k * V + j;
        y[i] = g[i] = xh[i] = v[j] = 0.f;
        a[i] = 1.f;
      }
      if (p.y) st.read(at, 3, k, yr(cur), left, nthV, y + k * V);
      if (GATE) st.read(at, 4, k, ur(cur), left, nthV, da + k * V);
      if (p.gx) st.read(at, 0, k, gxr(cur), left, nthV, g + k * V);
      if (p.gn) {
        st.read(at, 1, k, gnr(cur), left, nthV, v);
        st.read(at, 2, k, xr(cur), left, nthV, xh + k * V);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = k * V + j;
        y[i] *= ry;
        if (GATE) {
          const float u = da[i];
          float sg, so;
          sigmoid_pair<Accurate<T>::value>(u, sg, so);
          a[i] = KIND == GATE_SIGMOID ? sg : u * sg;
          da[i] = KIND == GATE_SIGMOID ? sg * so : sg * fmaf(u, so, 1.f);
        }
        const float c = ws[i] * a[i] * y[i];
        xh[i] = (xh[i] + c) * rx;               // rx = 0 without a next norm
        qn[i] = fmaf(v[j], xh[i], qn[i]);
        v[j] *= nw[i];
        g[i] = fmaf(rx, v[j], g[i]);
        sum[0] = fmaf(v[j], xh[i], sum[0]);
        sum[1] = fmaf(g[i], c, sum[1]);
        sum[2] = fmaf(xh[i], c, sum[2]);
      }
    }
    block_sum3(sum, red, slot);
    const float back = rx * (sum[0] * inv_n), s2 = (sum[1] - back * sum[2]) * inv_n;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      float oy[V], ou[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = k * V + j;
        g[i] = fmaf(-back, xh[i], g[i]);
        const float gw = g[i] * ws[i], gy = g[i] * y[i];
        q[i] = fmaf(gy, a[i], q[i]);
        ou[j] = GATE ? gw * y[i] * da[i] : 0.f;
        oy[j] = ry * fmaf(-y[i], s2, gw * a[i]);
      }
      if (k * nthV < left) {
        if (dx) store_vec<T, V>(dx + k * nthV, g + k * V);
        if (dy) store_vec<T, V>(dy + k * nthV, oy);
        if (GATE && du) store_vec<T, V>(du + k * nthV, ou);
      }
    }
    cur.next(gs, gt, gb, p.B);
  }
  st.wait(0);
  if (p.part) {
    float* o = p.part + (size_t)blockIdx.x * 2 * p.N;
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = c0 + k * nthV + j;
        if (c < p.N) {
          o[c] = q[k * V + j];
          o[p.N + c] = qn[k * V + j];
        }
      }
  }
}

// dw = scale Q, dscale = w Q (blockIdx.y = 0) and dw_next (1) from the blocks' partials: 32
// channels and 32 runs of blocks per thread block, summed in a fixed order.
static __global__ void __launch_bounds__(1024) k_norm_dw(int N, int blocks, const float* __restrict__ part,
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

// ---------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------
struct NormShape {
  int V, IT, threads;
  int grid;   // blocks launched, set by the launch
};
// the kernels of a direction, by element type (norm_fwd.cu, norm_bwd.cu)
int norm_run_forward(int dtype, const NormArgs& a, NormShape& s, int most, cudaStream_t st);
int norm_run_backward(int dtype, const NormArgs& a, NormShape& s, int most, cudaStream_t st);

}  // namespace delrec
