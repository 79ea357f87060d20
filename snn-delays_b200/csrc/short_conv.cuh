// Short causal convolution over time, one filter of K taps per channel, and its gradients:
//
//   p_t = b + sum_{d<K} w_{K-1-d} x_{t-d},    y_t = act(p_t),    act: identity or silu
//
// x_{-1} .. x_{-(K-1)} come from a state (K-1,B,N); a reset at t drops what lies before t.  A
// thread owns V neighbouring channels of one sequence and walks a chunk of time with the window
// (and, in the backward pass, the K partial sums of dx) in registers, so each tensor crosses the
// memory once apart from the K - 1 rows in front of (and behind) a chunk.
//
// What bounds it: latency, of loads that come a batch at a time to 13 to 18 warps an SM, and of the resets, a byte
// a row read within the row's work.  T=250 B=256 N=512 K=4 bf16: forward 42 us at 2.2 TB/s and 46 % of the issue
// slots, backward 77 us at 2.3 TB/s and 56 %; T=1021 B=24 N=700 K=3 fp32 with resets 25 and 42 us at 2.2 to 2.8 TB/s.
#pragma once

#include "seq_common.cuh"

namespace delrec {

enum { CONV_NONE = 0, CONV_SILU = 1 };
constexpr int kConvMaxK = 8;
constexpr int kConvAhead = 4;   // rows of x (and gy) on their way together; eight 16-bit ones of x alone

struct ConvArgs {
  int T, B, N, act, kind;       // kind of lengths: 0 int32, 1 int64, 2 one byte a row (0 or 1 steps)
  int chunks, steps;            // time is cut into chunks of `steps` rows
  const void *x, *state, *gy, *gs;
  const float *w, *bias;        // (N,K); (N) or NULL
  const void* lengths;
  const uint8_t* resets;
  void *y, *next, *dx, *ds;
  float* part;                  // (chunks * B, K + 1, N): partial sums of dw and db
  long long x_t, x_b, y_t, y_b, gy_t, gy_b, dx_t, dx_b;
};

__device__ __forceinline__ int conv_length(const ConvArgs& a, int b) {
  if (a.kind == 2) return a.lengths ? (((const uint8_t*)a.lengths)[b] ? a.T : 0) : a.T;
  return row_length(a.lengths, a.kind, b, a.T);
}

template <class T, int V>
__device__ __forceinline__ void conv_load(const T* ptr, float* v) {
  unpack_vec<T, V>(*(const VecOf<T, V>*)ptr, v);
}
template <class T, int V>
__device__ __forceinline__ void conv_store(T* ptr, const float* v) {
  *(VecOf<T, V>*)ptr = pack_vec<T, V>(v);
}

// y = silu(p) and its derivative
template <class T>
__device__ __forceinline__ float silu(float p, float& d) {
  float s, o;
  sigmoid_pair<false>(p, s, o);   // (one ex2: |p| 2^-24 of it, also in float32)
  d = s * fmaf(p, o, 1.f);
  return p * s;
}

// What a thread's filter and window have in common in both passes
template <class T, int K, int V>
struct ConvThread {
  const ConvArgs& a;
  int n, b, c, t0, t1, len;
  float w[K][V], bias[V], win[K > 1 ? K - 1 : 1][V];

  __device__ __forceinline__ ConvThread(const ConvArgs& a_) : a(a_) {}
  // false: no such thread
  __device__ __forceinline__ bool init() {
    const long long cols = (a.N + V - 1) / V;
    const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
    if (i >= cols * a.B * a.chunks) return false;
    n = (int)(i % cols) * V;
    const long long r = i / cols;
    b = (int)(r % a.B);
    c = (int)(r / a.B);
    t0 = c * a.steps;
    t1 = min(a.T, t0 + a.steps);
    len = conv_length(a, b);
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][v] = a.w[(size_t)(n + v) * K + k];
      bias[v] = a.bias ? a.bias[n + v] : 0.f;
    }
    return true;
  }
  __device__ __forceinline__ const T* row(const void* base, int t, long long st, long long sb) const {
    return (const T*)base + t * st + b * sb + n;
  }
  __device__ __forceinline__ size_t state_at(int j) const { return ((size_t)j * a.B + b) * a.N + n; }
  __device__ __forceinline__ bool cut(int t) const { return a.resets && a.resets[(size_t)t * a.B + b]; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j + 1 < K; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) win[j][v] = 0.f;
  }
  // win[j] is the input K - 1 - j steps back
  __device__ __forceinline__ void push(const float* x) {
#pragma unroll
    for (int j = 0; j + 2 < K; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) win[j][v] = win[j + 1][v];
    if (K > 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) win[K > 1 ? K - 2 : 0][v] = x[v];
    }
  }
  // the window in front of row t0 (t0 <= len)
  __device__ __forceinline__ void fill() {
    clear();
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) {
      const int t = t0 - (K - 1) + j;
      float x[V] = {};
      if (t < 0) {
        if (a.state) conv_load<T, V>((const T*)a.state + state_at(K - 1 + t), x);
      } else {
        if (cut(t)) clear();
        conv_load<T, V>(row(a.x, t, a.x_t, a.x_b), x);
      }
      push(x);
    }
  }
  __device__ __forceinline__ void pre(const float* x, float* p) const {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      p[v] = bias[v];
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) p[v] = fmaf(w[j][v], win[j][v], p[v]);
      p[v] = fmaf(w[K - 1][v], x[v], p[v]);
    }
  }
};

template <class T, int K, int V>
__global__ void __launch_bounds__(128, K <= 4 ? 6 : 4) k_conv_fwd(const ConvArgs a) {
  constexpr int AHEAD = sizeof(T) == 2 ? 2 * kConvAhead : kConvAhead;
  ConvThread<T, K, V> s(a);
  if (!s.init()) return;
  const int end = min(s.t1, s.len);
  const T* px = s.row(a.x, s.t0, a.x_t, a.x_b);
  T* py = const_cast<T*>(s.row(a.y, s.t0, a.y_t, a.y_b));
  using Row = VecOf<T, V>;
  const auto one = [&](int t, const Row& in, T* to) {
    float x[V], p[V];
    unpack_vec<T, V>(in, x);
    if (s.cut(t)) s.clear();
    s.pre(x, p);
    if (a.act == CONV_SILU) {
      float d;
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = silu<T>(p[v], d);
    }
    conv_store<T, V>(to, p);
    s.push(x);
  };
  int t = s.t0;
  if (t <= s.len) s.fill();
  for (; t + AHEAD <= end; t += AHEAD) {
    Row in[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) in[i] = *(const Row*)(px + i * a.x_t);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) one(t + i, in[i], py + i * a.y_t);
    px += AHEAD * a.x_t;
    py += AHEAD * a.y_t;
  }
  for (; t < end; ++t, px += a.x_t, py += a.y_t) one(t, *(const Row*)px, py);
  const float zero[V] = {};
  for (int t = max(s.t0, end); t < s.t1; ++t) conv_store<T, V>(const_cast<T*>(s.row(a.y, t, a.y_t, a.y_b)), zero);
  // the chunk that holds the last row there is writes the state behind it (chunk 0 of an empty sequence)
  if (K > 1 && a.next && s.c == max(s.len - 1, 0) / a.steps) {
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) conv_store<T, V>((T*)a.next + s.state_at(j), s.win[j]);
  }
}

// One row (T = 1, no resets): everything that a thread reads for a sequence is on its way at once, so that
// it takes one trip to the memory, and its filters serve every `step`-th sequence.  K = 4, in a graph, against
// the walk above: 256 x 512 bf16 4.1 -> 3.0 us (fp32 3.5 -> 3.1), 4096 x 512 bf16 24.5 -> 9.9.
template <class T, int K, int V>
__global__ void __launch_bounds__(128) k_conv_step(const ConvArgs a, int step) {
  const long long cols = (a.N + V - 1) / V, i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (i >= cols * step) return;
  const int n = (int)(i % cols) * V;
  using Row = VecOf<T, V>;
  float w[K * V], bias[V];
  if (V == 4) {
#pragma unroll
    for (int k = 0; k < K * V; k += 4) conv_load<float, 4>(a.w + (size_t)n * K + k, w + k);
  } else {
#pragma unroll
    for (int k = 0; k < K * V; ++k) w[k] = a.w[(size_t)n * K + k];
  }
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[n + v] : 0.f;
#pragma unroll 2
  for (long long b = i / cols; b < a.B; b += step) {
    const auto at = [&](int j) { return ((size_t)j * a.B + b) * a.N + n; };
    Row win[K] = {};
#pragma unroll
    for (int j = 0; j + 1 < K; ++j)
      if (a.state) win[j] = *(const Row*)((const T*)a.state + at(j));
    const bool live = conv_length(a, (int)b) > 0;
    if (live) win[K - 1] = *(const Row*)((const T*)a.x + b * a.x_b + n);   // what does not count is not read
    float p[V];
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = bias[v];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      float x[V];
      unpack_vec<T, V>(win[j], x);
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = fmaf(w[v * K + j], x[v], p[v]);
    }
    if (a.act == CONV_SILU) {
      float d;
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = silu<T>(p[v], d);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = live ? p[v] : 0.f;
    conv_store<T, V>((T*)a.y + b * a.y_b + n, p);
    if (a.next) {
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) *(Row*)((T*)a.next + at(j)) = live ? win[j + 1] : win[j];
    }
  }
}

// One walk forward: p_t from the window, dp_t = gy_t act'(p_t), which adds to the dx of the K
// positions t - d (acc[d]; those behind a reset take no more), to dw and to db.  Position t - K + 1
// is then complete.  A chunk walks K - 1 rows into the next one for its last positions and counts
// dw and db of its own rows only.
template <class T, int K, int V>
__global__ void __launch_bounds__(128) k_conv_bwd(const ConvArgs a) {
  ConvThread<T, K, V> s(a);
  if (!s.init()) return;
  float acc[K][V], dw[K][V], db[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    db[v] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) acc[k][v] = dw[k][v] = 0.f;
  }
  // rows since the last reset: a row reaches the positions at most that far back
  int since = 1 << 30;
  const int end = min(s.t1 + K - 1, s.len);
  // position pos >= 0 of dx, or of the state's gradient
  const auto emit = [&](int pos, const float* g) {
    if (pos >= 0) {
      if (pos >= s.t0 && pos < s.t1 && a.dx) conv_store<T, V>(const_cast<T*>(s.row(a.dx, pos, a.dx_t, a.dx_b)), g);
    } else if (s.c == 0 && pos >= 1 - K && a.ds) {
      conv_store<T, V>((T*)a.ds + s.state_at(K - 1 + pos), g);
    }
  };
  if (s.t0 <= s.len) {
    const T *px = s.row(a.x, s.t0, a.x_t, a.x_b), *pg = a.gy ? s.row(a.gy, s.t0, a.gy_t, a.gy_b) : nullptr;
    using Row = VecOf<T, V>;
    s.fill();
    const auto one = [&](int t, const Row& in, const Row& gin) {
      float x[V], g[V];
      unpack_vec<T, V>(in, x);
      unpack_vec<T, V>(gin, g);
      since = min(since + 1, 1 << 30);
      if (s.cut(t)) {
        s.clear();
        since = 0;
      }
      if (a.act == CONV_SILU) {
        float p[V], d;
        s.pre(x, p);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          silu<T>(p[v], d);
          g[v] *= d;
        }
      }
#pragma unroll
      for (int d = 0; d < K; ++d)
        if (d <= since) {
#pragma unroll
          for (int v = 0; v < V; ++v) acc[d][v] = fmaf(s.w[K - 1 - d][v], g[v], acc[d][v]);
        }
      if (t < s.t1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          db[v] += g[v];
          dw[K - 1][v] = fmaf(g[v], x[v], dw[K - 1][v]);
#pragma unroll
          for (int j = 0; j + 1 < K; ++j) dw[j][v] = fmaf(g[v], s.win[j][v], dw[j][v]);
        }
      }
      emit(t - (K - 1), acc[K - 1]);
      s.push(x);
#pragma unroll
      for (int d = K - 1; d > 0; --d)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[d][v] = acc[d - 1][v];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[0][v] = 0.f;
    };
    int t = s.t0;
    for (; t + kConvAhead <= end; t += kConvAhead) {
      Row in[kConvAhead], gin[kConvAhead];
#pragma unroll
      for (int i = 0; i < kConvAhead; ++i) {
        in[i] = *(const Row*)(px + i * a.x_t);
        gin[i] = pg ? *(const Row*)(pg + i * a.gy_t) : Row{};
      }
      px += kConvAhead * a.x_t;
      if (pg) pg += kConvAhead * a.gy_t;
#pragma unroll
      for (int i = 0; i < kConvAhead; ++i) one(t + i, in[i], gin[i]);
    }
    for (; t < end; ++t, px += a.x_t) {
      one(t, *(const Row*)px, pg ? *(const Row*)pg : Row{});
      if (pg) pg += a.gy_t;
    }
    // acc[d] now belongs to position last - d + 1, last the last row walked; those of the new state
    // take its gradient
    const int last = max(end, s.t0) - 1;
#pragma unroll
    for (int d = K - 1; d > 0; --d) {
      const int pos = last - d + 1, j = pos - (s.len - (K - 1));
      if (a.gs && j >= 0 && d - 1 <= since && last == s.len - 1) {
        float g[V];
        conv_load<T, V>((const T*)a.gs + s.state_at(j), g);
#pragma unroll
        for (int v = 0; v < V; ++v) acc[d][v] += g[v];
      }
      emit(pos, acc[d]);
    }
  }
  const float zero[V] = {};
  if (a.dx)
    for (int t = max(s.t0, s.len); t < s.t1; ++t)
      conv_store<T, V>(const_cast<T*>(s.row(a.dx, t, a.dx_t, a.dx_b)), zero);
  if (a.part) {
    float* q = a.part + ((size_t)s.c * a.B + s.b) * (K + 1) * a.N + s.n;
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) q[(size_t)k * a.N + v] = k < K ? dw[k < K ? k : 0][v] : db[v];
  }
}

// dw (N,K) and db (N): the partial sums in the order of (chunk, sequence), in 64 bits (the kernel waits for its reads:
// the same time, and 1.9e-7 -> 1.4e-7 off at T=1021 B=24 N=700 fp32).  Block: 32 channels of one tap by 32 runs of parts.
static __global__ void __launch_bounds__(1024) k_conv_dw(int N, int K, int parts, const float* __restrict__ part,
                                                  float* __restrict__ dw, float* __restrict__ db) {
  __shared__ double sum[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, n = blockIdx.x * 32 + lane, k = blockIdx.y;
  const int p0 = (int)((long long)parts * run / 32), p1 = (int)((long long)parts * (run + 1) / 32);
  double s = 0.0;
  if (n < N)
    for (int p = p0; p < p1; ++p) s += part[((size_t)p * (K + 1) + k) * N + n];
  sum[run][lane] = s;
  __syncthreads();
  if (run == 0 && n < N) {
    double t = 0.0;
    for (int r = 0; r < 32; ++r) t += sum[r][lane];
    if (k < K) {
      if (dw) dw[(size_t)n * K + k] = (float)t;
    } else if (db) {
      db[n] = (float)t;
    }
  }
}

}  // namespace delrec
