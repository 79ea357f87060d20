// The vocabulary losses' kernels around their matrix products (vocab_gemm.cuh).  Rows (positions) that
// do not count are packed away first: the products run over the others only, and what stands in a
// padded position is not read.
//
//   loss_m = tau^2 sum_k p_k (log p_k - log q_{i_k}),  q = softmax((x W^T + b) / tau)
//   d loss_m / d z_v = tau (q_v - sum_{k: i_k = v} p_k)
//
// p = softmax(t / tau) over the K kept logits t of a teacher; the cross entropy is K = 1, p = 1,
// tau = 1.  Exponentials are of y = z log2(e) / tau, sums in float32.
#pragma once

#include "seq_common.cuh"

namespace delrec {

constexpr int kVocabMaxD = 8192, kVocabMaxK = 1024;
constexpr float kLn2v = 0.6931471805599453f;
constexpr int kVocabIndexRange = 1 << 1;   // ST_INDEX_RANGE of the status word

struct VocabArgs {
  int T, B, D, V, K, M;            // M = T B positions
  int distill, wide, index_wide, teacher;   // types of lengths, indices and the teacher's logits
  long long ignore;
  float tau, scale;                // scale = log2(e) / tau
  long long x_t, x_b;
  const void *x, *w, *bias, *index, *logits, *lengths;
  uint8_t* flags;                  // (M) distillation: does the position count
  int *rows, *rowmap, *pos;        // count; position of each packed row; packed row of each position or -1
  int* idx;                        // (M, K) of packed rows: tokens in rising order, each once, then -1
  float *p, *y, *h, *lse, *loss;   // p (NULL for K = 1: 1) and y (M, K): z, then log2 q; h, lse, loss (M): of packed rows
  int* ticket;                     // blocks that are done with their rows' losses
  int* status;
};

__device__ __forceinline__ long long vocab_index(const VocabArgs& a, size_t i) {
  return a.index_wide ? ((const long long*)a.index)[i] : (long long)((const int*)a.index)[i];
}
__device__ __forceinline__ float vocab_teacher(const VocabArgs& a, size_t i) {
  switch (a.teacher) {
    case DELREC_F32: return ((const float*)a.logits)[i];
    case DELREC_BF16: return to_f(((const __nv_bfloat16*)a.logits)[i]);
  }
  return to_f(((const __half*)a.logits)[i]);
}
__device__ __forceinline__ bool vocab_live(const VocabArgs& a, int m) {
  return !a.lengths || m / a.B < row_length(a.lengths, a.wide, m % a.B, a.T);
}
// a kept entry of the teacher's list
__device__ __forceinline__ bool vocab_kept(long long i, float t) { return i >= 0 && t != -INFINITY; }

// distillation: a position counts if its list keeps an entry.  One warp a position.
static __global__ void __launch_bounds__(256) k_vocab_flags(const VocabArgs a) {
  const int m = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (m >= a.M) return;
  bool any = false;
  if (vocab_live(a, m))
    for (int k = lane; k < a.K; k += 32)
      any |= vocab_kept(vocab_index(a, (size_t)m * a.K + k), vocab_teacher(a, (size_t)m * a.K + k));
  any = __any_sync(0xffffffffu, any);
  if (lane == 0) a.flags[m] = any;
}
__device__ __forceinline__ bool vocab_counts(const VocabArgs& a, int m) {
  if (a.distill) return a.flags[m];
  return vocab_live(a, m) && vocab_index(a, m) != a.ignore;
}
// rows that count in each block of 1024
static __global__ void __launch_bounds__(1024) k_vocab_count(const VocabArgs a, int* counts) {
  const int m = blockIdx.x * 1024 + threadIdx.x;
  const int n = __syncthreads_count(m < a.M && vocab_counts(a, m));
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}
// Packs the rows that count, in order.  A block of 1024 counts those before its own by itself, from the
// blocks' counts where those are given.  each (M) or NULL: the positions' losses, 0 where a position does
// not count.
static __global__ void __launch_bounds__(1024) k_vocab_rows(const VocabArgs a, const int* __restrict__ counts, float* each) {
  __shared__ int s_warp[32], s_before;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, first = blockIdx.x * 1024;
  int before = 0;
  if (counts) {
    for (int k = tid; k < (int)blockIdx.x; k += 1024) before += counts[k];
  } else {
#pragma unroll 4
    for (int m = tid; m < first; m += 1024) before += vocab_counts(a, m);
  }
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) s_warp[warp] = before;
  __syncthreads();
  if (warp == 0) {
    const int v = __reduce_add_sync(0xffffffffu, s_warp[lane]);
    if (lane == 0) s_before = v;
  }
  __syncthreads();
  const int m = first + tid;
  const bool on = m < a.M && vocab_counts(a, m);
  const unsigned vote = __ballot_sync(0xffffffffu, on);
  if (lane == 0) s_warp[warp] = __popc(vote);
  __syncthreads();
  int at = s_before, total = s_before;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) at += s_warp[w];
    total += s_warp[w];
  }
  at += __popc(vote & ((1u << lane) - 1u));
  if (m < a.M) {
    a.pos[m] = on ? at : -1;
    if (on) a.rowmap[at] = m;
    else if (each) each[m] = 0.f;
  }
  if (tid == 0 && first + 1024 >= a.M) {
    *a.rows = total;
    *a.ticket = 0;
  }
}

// Rows as tensor-core operands: out[piece][row][Dp], 16-bit types as they are, fp32 in three bf16 pieces
// (v = p0 + p1 + p2 exactly).  rows NULL: n rows in place, else the packed rows of x and zero rows up to
// the next 64.  A thread takes eight columns.
struct VocabPack {
  const void* src;
  long long st, sb, n, piece;
  int B, D, Dp, vec;               // vec: 16 bytes of a row at a time
  const int *rows, *rowmap;
  void* out;
};
template <class T>
__device__ __forceinline__ void vocab_pack(const VocabPack& k_, long long first, long long step) {
  const T* src = (const T*)k_.src;
  const int *rows = k_.rows, *rowmap = k_.rowmap, B = k_.B, D = k_.D, Dp = k_.Dp;
  const long long n = k_.n, st = k_.st, sb = k_.sb, piece = k_.piece;
  const int cols = Dp / 8;
  const long long real = rows ? *rows : n, all = (rows ? (real + 63) / 64 * 64 : n) * cols;
  for (long long i = first; i < all; i += step) {
    const long long r = i / cols;
    const int c = (int)(i % cols) * 8;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
    if (r < real) {
      const long long m = rows ? rowmap[r] : r;
      const T* s = src + (rows ? m / B * st + m % B * sb : m * st) + c;
      if (k_.vec && c + 8 <= D) {
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8; k += W) unpack_vec<T, W>(*(const VecOf<T, W>*)(s + k), v + k);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < D) v[k] = to_f(s[k]);
      }
    }
    using E = std::conditional_t<std::is_same_v<T, __half>, __half, __nv_bfloat16>;
    E* o = (E*)k_.out + r * Dp + c;
    constexpr int P = sizeof(T) == 4 ? 3 : 1;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const VecOf<E, 8> q = pack_vec<E, 8>(v);
      *(VecOf<E, 8>*)(o + p * piece) = q;
      if (p + 1 < P) {
        float f[8];
        unpack_vec<E, 8>(q, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] -= f[k];
      }
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) k_vocab_pack(const VocabPack k) {
  vocab_pack<T>(k, blockIdx.x * 256LL + threadIdx.x, gridDim.x * 256LL);
}

// entry e of a teacher's lists, `there` if it is one: its token and logit, kVocabNone and -inf where it is left out,
// kVocabNone and bad where its index is past the vocabulary
constexpr int kVocabNone = 0x7fffffff;
__device__ __forceinline__ int vocab_entry(const VocabArgs& a, size_t e, bool there, float& t, bool& bad) {
  t = -INFINITY;
  if (!there) return kVocabNone;
  const long long i = vocab_index(a, e);
  const float v = vocab_teacher(a, e);
  if (!vocab_kept(i, v)) return kVocabNone;
  t = v;
  if (i < a.V) return (int)i;
  atomicOr(a.status, kVocabIndexRange);
  bad = true;
  return kVocabNone;
}
// where each half tile of `cols` columns finds its first of the n tokens of a rising list, by `step` threads
__device__ __forceinline__ void vocab_halves(const int* list, int n, int first, int step, unsigned* tab, long long ld, int halves,
                                             int cols) {
  for (int t = first; t < halves; t += step) {
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (list[mid] < t * cols) lo = mid + 1;
      else hi = mid;
    }
    const int off = lo < n ? list[lo] - t * cols : cols;
    tab[t * ld] = (unsigned)lo << 8 | (off < cols ? off : 255);
  }
}

// The targets of a packed row: their tokens in rising order, each once, with the sum of its p (then -1), h = sum p log p,
// and where each half tile of the logits (`cols` columns) finds its first target: tab[half][row] = place in the list << 8 |
// column, 255 without one (tab NULL: not wanted).  Differences of a teacher's logits are taken first: those of the
// type's lowest value stay finite at any temperature.
//
// Their logits come from the product that makes the statistics: a dot product of its own is off by another rounding
// than the log-sum-exp (the tensor core's accumulator truncates), and that difference is all there is of the loss of a
// target that is nearly certain (z = 40 over 512 channels: -4e-5 of 0).  It takes longer, too (4096 rows on 32768 tokens, 512
// channels, bf16, forward: 64 targets 171 us instead of 154, 1024 targets 1573 instead of 414).
//
// W threads to a row: one for one target; a warp, an entry to a lane, up to 32 (sorted by counting, K steps: 4096 rows of
// four 22 us of the small pass, 26 by the block's way); else a block, by a bitonic sort of P places (K's power of two, 128
// at least).  The blocks from `blocks` on bring x into operands: both wait for the packed rows alone.
template <class T, int W>
__global__ void __launch_bounds__(128) k_vocab_targets(const VocabArgs a, int blocks, const VocabPack pack, unsigned* tab,
                                                       long long ld, int halves, int cols, int P) {
  if ((int)blockIdx.x >= blocks) {
    vocab_pack<T>(pack, (blockIdx.x - blocks) * 128LL + threadIdx.x, (gridDim.x - blocks) * 128LL);
    return;
  }
  const int r = blockIdx.x * (128 / W) + threadIdx.x / W;
  if (r >= *a.rows) return;        // whole warps with W = 32, the whole block with W = 128
  const int m = a.rowmap[r], K = a.K;
  if constexpr (W == 1) {          // K = 1: p = 1
    const long long i = vocab_index(a, m);
    const bool in = i >= 0 && i < a.V, ok = in && (!a.distill || fabsf(vocab_teacher(a, m)) < INFINITY);
    if (!in) atomicOr(a.status, kVocabIndexRange);
    a.idx[r] = ok ? (int)i : -1;
    if (!ok) a.y[r] = __int_as_float(0x7fc00000);
  } else if constexpr (W == 32) {  // an entry to a lane
    __shared__ int s_few[4][32];
    constexpr unsigned full = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    const auto all = [&](float v, bool max) {
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const float u = __shfl_xor_sync(full, v, o);
        v = max ? fmaxf(v, u) : v + u;
      }
      return v;
    };
    bool bad = false;
    float t;
    const int i = vocab_entry(a, (size_t)m * K + lane, lane < K, t, bad);
    const float top = all(t, true), sum = all(t == -INFINITY ? 0.f : expf((t - top) / a.tau), false);
    const float lp = (t - top) / a.tau - logf(sum), p = t == -INFINITY ? 0.f : expf(lp);
    const float h = all(bad ? __int_as_float(0x7fc00000) : p != 0.f ? p * lp : 0.f, false);
    if (lane == 0) a.h[r] = h;
    float s = 0.f;
    int first = 32, rank = 0;
    for (int j = K - 1; j >= 0; --j) {
      const float q = __shfl_sync(full, p, j);
      if (__shfl_sync(full, i, j) == i) {
        s += q;
        first = j;
      }
    }
    const bool on = i != kVocabNone && first == lane;
    const int u = on ? i : kVocabNone, n = __popc(__ballot_sync(full, on));
    for (int j = 0; j < K; ++j) rank += __shfl_sync(full, u, j) < i;
    const size_t e = (size_t)r * K;
    if (on) {
      a.idx[e + rank] = i;
      a.p[e + rank] = s;
    }
    if (lane >= n && lane < K) {
      a.idx[e + lane] = -1;
      a.p[e + lane] = a.y[e + lane] = 0.f;
    }
    if (!tab) return;
    int* s_i = s_few[threadIdx.x >> 5];
    if (on) s_i[rank] = i;
    __syncwarp();
    vocab_halves(s_i, n, lane, 32, tab + r, ld, halves, cols);
  } else {
    extern __shared__ unsigned long long s_key[];    // [P] token and place, in rising order
    __shared__ float s_red[4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* s_p = (float*)(s_key + P);                // [P]
    int* s_i = (int*)(s_p + P);                      // [P] the tokens, each once
    const auto token = [&](int e) { return (int)(s_key[e] >> 10); };
    const auto all = [&](float v, bool max) {
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = max ? fmaxf(v, u) : v + u;
      }
      __syncthreads();
      if (lane == 0) s_red[warp] = v;
      __syncthreads();
      v = s_red[0];
      for (int w = 1; w < 4; ++w) v = max ? fmaxf(v, s_red[w]) : v + s_red[w];
      return v;
    };
    float top = -INFINITY, h = 0.f;
    for (int k = tid; k < P; k += W) {
      bool bad = false;
      float t;
      const int i = vocab_entry(a, (size_t)m * K + k, k < K, t, bad);
      if (bad) h = __int_as_float(0x7fc00000);
      s_key[k] = (unsigned long long)i << 10 | k;
      s_p[k] = t;
      top = fmaxf(top, t);
    }
    top = all(top, true);
    float sum = 0.f;
    for (int k = tid; k < K; k += W) sum += s_p[k] == -INFINITY ? 0.f : expf((s_p[k] - top) / a.tau);
    const float ls = logf(all(sum, false));
    for (int k = tid; k < K; k += W) {
      const float lp = (s_p[k] - top) / a.tau - ls, p = s_p[k] == -INFINITY ? 0.f : expf(lp);
      s_p[k] = p;
      if (p != 0.f) h = fmaf(p, lp, h);
    }
    h = all(h, false);
    if (tid == 0) a.h[r] = h;
    __syncthreads();
    for (int size = 2; size <= P; size *= 2)         // bitonic sort
      for (int step = size / 2; step; step /= 2) {
        for (int j = tid; j < P / 2; j += W) {
          const int lo = 2 * j - (j & (step - 1)), hi = lo + step;
          const unsigned long long u = s_key[lo], v = s_key[hi];
          if ((u > v) == !(lo & size)) {
            s_key[lo] = v;
            s_key[hi] = u;
          }
        }
        __syncthreads();
      }
    // a thread's stretch of the sorted list: its tokens that stand there first, behind those of the threads before
    const int C = P / W, e0 = tid * C;
    int before = e0 ? token(e0 - 1) : kVocabNone, own = 0;
    for (int e = e0; e < e0 + C; ++e) {
      const int i = token(e);
      own += i != kVocabNone && i != before;
      before = i;
    }
    int at = own, n = 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += u;
    }
    __syncthreads();
    if (lane == 31) s_red[warp] = __int_as_float(at);
    __syncthreads();
    at -= own;
    for (int w = 0; w < 4; ++w) {
      const int u = __float_as_int(s_red[w]);
      at += w < warp ? u : 0;
      n += u;
    }
    before = e0 ? token(e0 - 1) : kVocabNone;
    for (int e = e0; e < e0 + C; ++e) {
      const int i = token(e);
      if (i != kVocabNone && i != before) {
        float s = 0.f;
        for (int j = e; j < P && token(j) == i; ++j) s += s_p[s_key[j] & 1023];
        s_i[at] = i;
        a.idx[(size_t)r * K + at] = i;
        a.p[(size_t)r * K + at] = s;
        ++at;
      }
      before = i;
    }
    for (int k = n + tid; k < K; k += W) {
      a.idx[(size_t)r * K + k] = -1;
      a.p[(size_t)r * K + k] = a.y[(size_t)r * K + k] = 0.f;
    }
    __syncthreads();
    vocab_halves(s_i, n, tid, W, tab + r, ld, halves, cols);
  }
}

// A row's log-sum-exp from its tiles' maxima and sums, and its loss.  Block: 32 rows by 32 runs of tiles.
__device__ __forceinline__ void vocab_join(float& top, float& sum, float2 v) {
  const float mx = fmaxf(top, v.x), at = mx == -INFINITY ? 0.f : mx;
  sum = sum * exp2f(top - at) + v.y * exp2f(v.x - at);
  top = mx;
}
// The targets' logits in y become d = log2 q, from the row's maximum and sum themselves: a loss near 0 keeps
// its sign, and is off by what the sum's 1 is off.  A warp to a row's targets.
// out not NULL: the block that comes last adds the rows' losses up, in a fixed order (their mean: divided;
// 0 of none).
static __global__ void __launch_bounds__(1024) k_vocab_lse(const VocabArgs a, const float2* __restrict__ part,
                                                           long long ld, int tiles, float* each, int mean, float* out) {
  __shared__ float2 s[32][33];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int rows = *a.rows, r = blockIdx.x * 32 + lane, used = max((rows + 31) / 32, 1);
  if ((int)blockIdx.x >= used) return;
  float top = -INFINITY, sum = 0.f;
  if (r < rows)
    for (int t0 = run; t0 < tiles; t0 += 32 * 8) {
      float2 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = t0 + 32 * k < tiles ? part[(t0 + 32 * k) * ld + r] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) vocab_join(top, sum, v[k]);
    }
  s[run][lane] = make_float2(top, sum);
  __syncthreads();
  for (int k = 16; k; k >>= 1) {
    if (run < k) {
      vocab_join(top, sum, s[run + k][lane]);
      s[run][lane] = make_float2(top, sum);
    }
    __syncthreads();
  }
  const int mine = blockIdx.x * 32 + run;
  if (mine < rows) {
    top = s[0][run].x;
    const float ls = log2f(s[0][run].y);
    float dot = 0.f;
    for (int k = lane; k < a.K; k += 32) {
      const size_t e = (size_t)mine * a.K + k;
      const float z = a.y[e];
      float d = fmaf(z, a.scale, -top) - ls;
      d = d > 0.f ? 0.f : d;            // (NaN stays)
      a.y[e] = d;
      const float p = a.p ? a.p[e] : 1.f;
      // a logit that a mask made the type's lowest value has no z log2(e), but a loss
      if (p != 0.f) dot = fmaf(p, d == -INFINITY && z > -INFINITY ? z / a.tau : kLn2v * d, dot);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == 0) {
      a.lse[mine] = top + ls;
      const float loss = a.tau * a.tau * ((a.p ? a.h[mine] : 0.f) - dot);
      a.loss[mine] = loss;
      if (each) each[a.rowmap[mine]] = loss;
    }
  }
  if (!out) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(a.ticket, 1) == used - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double* total = (double*)s;
  double v = 0.0;
#pragma unroll 4
  for (int k = threadIdx.x; k < rows; k += 1024) v += __ldcg(a.loss + k);
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) total[run] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0.0;
    for (int w = 0; w < 32; ++w) v += total[w];
    *out = (float)(mean && rows > 0 ? v / rows : v);
  }
}

// c_r = g tau (/ count) of each packed row in G = c (q - p), times a power of two whose inverse goes into
// *inv: at most 2^14, so that G fits fp16 with its small entries.  Where all rows share one c, c itself
// goes into *inv: c (q - 1) of a small q would round alike in every row, up to half a step off in a 16-bit
// type (8192 positions on 32768 tokens bf16: gradients 3.3e-3 -> 1.7e-3 off, as much as the result's own
// rounding).  A row with a NaN loss has NaN gradients.
static __global__ void __launch_bounds__(1024) k_vocab_coef(const VocabArgs a, int reduction, const float* __restrict__ g,
                                                            float* coef, float* inv) {
  __shared__ float s_top[32];
  const int rows = *a.rows, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (reduction != 0) {
#pragma unroll 4
    for (int r = threadIdx.x; r < rows; r += 1024) {
      const float l = a.loss[r];
      coef[r] = l != l ? l : 16384.f;
    }
    // (nothing counts: gradients of 0 whatever *g is)
    if (threadIdx.x == 0) *inv = rows ? *g * a.tau / (reduction == 1 ? (float)rows : 1.f) * (1.f / 16384.f) : 0.f;
    return;
  }
  float top = 0.f;
#pragma unroll 4
  for (int r = threadIdx.x; r < rows; r += 1024) {
    const float c = fabsf(g[a.rowmap[r]] * a.tau);
    if (c < INFINITY) top = fmaxf(top, c);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  for (int w = 0; w < 32; ++w) top = fmaxf(top, s_top[w]);
  int e = 0;
  frexpf(top, &e);                                        // top = f 2^e, f in [0.5, 1)
  e = top > 0.f ? min(max(14 - e, -100), 120) : 0;
  const float up = ldexpf(1.f, e);
#pragma unroll 4
  for (int r = threadIdx.x; r < rows; r += 1024) {
    const float c = g[a.rowmap[r]] * a.tau, l = a.loss[r];
    coef[r] = l != l ? l : c * up;
  }
  if (threadIdx.x == 0) *inv = ldexpf(1.f, -e);
}

// the targets' entries of a piece of G: c (q - p), each rounded once; near q = p = 1 from what is left of them
template <class E>
__global__ void __launch_bounds__(256) k_vocab_patch(const VocabArgs a, const float* __restrict__ coef, int v0, int n,
                                                     E* G, long long ld, long long piece, int pieces) {
  const long long e = blockIdx.x * 256LL + threadIdx.x;
  const long long r = e / a.K;
  if (r >= *a.rows) return;
  const int i = a.idx[e] - v0;
  if (i < 0 || i >= n) return;
  const float d = a.y[e], t = a.p ? a.p[e] : 1.f;
  float v = coef[r] * (t > 0.5f ? expm1f(kLn2v * d) + (1.f - t) : exp2f(d) - t);
  for (int p = 0; p < pieces; ++p) {
    const E q = from_f<E>(v);
    G[p * piece + r * ld + i] = q;
    v -= to_f(q);
  }
}

// column sums of a piece of G over runs of rows: part[run][column]; then db.  Eight columns a thread (a
// row's pitch is a multiple of 256).
template <class E, int P>
__global__ void __launch_bounds__(128) k_vocab_db_part(const int* __restrict__ rows, const E* __restrict__ G, int n,
                                                       long long ld, long long piece, float* part) {
  const int c = (blockIdx.x * 128 + threadIdx.x) * 8, run = blockIdx.y, runs = gridDim.y;
  if (c >= n) return;
  const long long R = *rows, r0 = R * run / runs, r1 = R * (run + 1) / runs;
  float s[8] = {};
#pragma unroll 4
  for (long long r = r0; r < r1; ++r) {
    float v[8], f[8];
    unpack_vec<E, 8>(*(const VecOf<E, 8>*)(G + r * ld + c), v);
#pragma unroll
    for (int p = 1; p < P; ++p) {
      unpack_vec<E, 8>(*(const VecOf<E, 8>*)(G + p * piece + r * ld + c), f);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += f[k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] += v[k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (c + k < n) part[(long long)run * n + c + k] = s[k];
}
template <class T>
__global__ void __launch_bounds__(256) k_vocab_db(const float* __restrict__ part, int n, int runs,
                                                  const float* __restrict__ inv, T* db) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float s = 0.f;
  for (int k = 0; k < runs; ++k) s += part[(long long)k * n + c];
  db[c] = from_f<T>(s * *inv);
}

// out[row][D] = *inv * sum of planes[split][pos ? pos[row] : row], 0 where pos is -1
template <class T>
__global__ void __launch_bounds__(256) k_vocab_planes(long long n, int D, const int* __restrict__ pos,
                                                      const float* __restrict__ plane, long long ld, long long split,
                                                      int splits, const float* __restrict__ inv, T* out) {
  const int cols = (D + 3) / 4;
  const float up = *inv;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n * cols; i += gridDim.x * 256LL) {
    const long long m = i / cols, r = pos ? pos[m] : m;
    const int c = (int)(i % cols) * 4;
    float v[4] = {};
    if (r >= 0)
      for (int s = 0; s < splits; ++s) {
        const float4 q = *(const float4*)(plane + s * split + r * ld + c);
        v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
      }
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = r >= 0 ? v[k] * up : 0.f;   // 0 where a position does not count, also of an infinite up
    T* o = out + m * D + c;
    if (D % 4 == 0) {
      *(VecOf<T, 4>*)o = pack_vec<T, 4>(v);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < D) o[k] = from_f<T>(v[k]);
    }
  }
}

}  // namespace delrec
