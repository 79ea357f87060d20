// Tensor-core products of the vocabulary losses (tcgen05 + TMA + tensor memory), fused with what
// follows them:
//
//   logits      z = x W^T (rows x vocabulary), never stored.  VG_STATS: each row's maximum and sum of
//               exponentials over the tile's columns, and the logits of its targets.  VG_GRAD:
//               c_m softmax(z)_mv in the operands' type, from the row's log-sum-exp, for one piece of the
//               vocabulary.
//   dW = G^T x  and  dx += G W  for that piece (VG_OUT).
//
// Persistent: a pair of CTAs on two SMs walks 256 x BN output tiles (cta_group::2).  Each keeps 128 rows
// of A and of the accumulators, and half of B's columns, which the tensor cores of both read: a 256 x 256
// tile's operands then take 32 instead of 48 KB a SM and 64-block (8192 positions on 32768 tokens, 512
// channels: the gradients' products 115 -> 99 us each).  The gradients' products take 512 columns to a
// tile (BN = 512, one accumulator) where those are there: 24 KB for as much work (training pass of the
// same 755 -> 718 us of backward).  In each CTA one thread streams operand tiles
// with TMA (no multicast) into a ring of shared-memory stages; in the first one a thread issues tcgen05.mma (M=256, N=BN, K=16)
// into one of two accumulators in tensor memory; eight warps of each read the other one back, so
// the epilogue of a tile runs under the next tile's products.  fp32 operands are three bf16 pieces each (an exact split) and six piece
// products, smallest first; 16-bit operands are taken as they are.  The tensor core's accumulator
// truncates, so fp32 reductions run in segments whose sums are added outside it: the logits' of 128
// columns, in registers, the gradients' of 512, in their result (2000 positions on 5003 tokens, 700 channels, off by 1.9e-6 -> 9e-7 in dx and
// 1.2e-6 -> 6e-7 in dweight, in the same time).
//
// The number of rows is read from the device (rows that do not count are packed away before).
// Every wait is bounded: on expiry the CTA records ST_TIMEOUT, drains its copies and returns.
#pragma once

#include "f32x2.cuh"
#include "seq_common.cuh"
#include "tc_ptx.cuh"

namespace delrec {

enum { VG_STATS = 0, VG_GRAD = 1, VG_OUT = 2 };
constexpr int kVgEpi = 8;             // epilogue warps
constexpr int kVgThreads = 32 * (kVgEpi + 2);   // then one for TMA, one for MMA
constexpr int kVgMaxProd = 6;
// Targets of a row up to which a tile looks through all of them (4096 positions of five on 32768 tokens: 119.7 us forward,
// by the table 124.2).
constexpr int kVgFew = 8;
constexpr int kVgTimeout = 1 << 3;    // ST_TIMEOUT of the status word

struct VgArgs {
  const int* rows;              // device: rows that count
  int M, K;                     // output rows and reduction length; -1: *rows
  int N;                        // output columns
  int nprod, pa[kVgMaxProd], pb[kVgMaxProd];
  int b_mn, b_k;                // where B starts
  int splits, seg;              // reduction in `splits` parts of whole segments of `seg` 64-blocks (0: one per part)
  int* status;
  long long spin_ns;
  // VG_STATS: part[2 * column tile + half][row] = {max, sum}, in units of log2
  float2* part;
  long long part_ld;
  // .. and the rows' targets: their columns in rising order (rows, kept), where a half tile's begin (see
  // k_vocab_targets; NULL for kept <= kVgFew), their logits
  const int* idx;
  const unsigned* tab;
  float* z;
  int kept;
  const void* bias;             // of the columns (element type), NULL: 0
  int bias_code;                // its element type
  float scale;                  // log2(e) / temperature
  // VG_GRAD: G (piece, row, column), pitch g_ld
  const float *lse, *coef;      // log2 of the sum of exponentials; c_m
  void* G;
  long long g_ld, g_piece;
  int pieces;
  // VG_OUT: planes (split, row, column) float32, or the result itself in the element type
  float* plane;
  long long plane_ld, plane_split;
  int accumulate;               // add to what the planes hold
  void* out;                    // not NULL: out[(out0 + row) * out_ld + column] = sum * *inv
  long long out_ld, out0;
  const float* inv;
};

constexpr int vg_stages(int BN) { return BN == 512 ? 4 : BN == 256 ? 6 : 8; }
constexpr size_t vg_smem(int BN) { return (size_t)vg_stages(BN) * (128 * 64 + BN / 2 * 64) * 2 + 1024; }

// bar: an mbarrier of the pair's first CTA
__device__ __forceinline__ void vg_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"((unsigned long long)map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// the address of the same place in the pair's first CTA
__device__ __forceinline__ uint32_t vg_first(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void vg_arrive(uint32_t bar) {   // a shared::cluster address
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void vg_mma(uint32_t tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(
          tmem),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
// arrives at this barrier of both CTAs once the products issued so far are done
__device__ __forceinline__ void vg_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((unsigned short)3)
               : "memory");
}
__device__ __forceinline__ void vg_meet() {   // both CTAs of the pair
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Waits at most limit_ns; false when the time is up here or was elsewhere in the CTA.
__device__ __forceinline__ bool vg_wait(uint32_t bar, uint32_t parity, long long limit_ns, volatile int* abort, int* status) {
  if (mbar_try(bar, parity)) return true;
  const unsigned long long t0 = global_ns();
  for (unsigned it = 1;; ++it) {
    if (mbar_try(bar, parity)) return true;
    if ((it & 63) == 0) {
      if (*abort) return false;
      if ((long long)(global_ns() - t0) > limit_ns) {
        *abort = 1;
        atomicOr(status, kVgTimeout);
        return false;
      }
    }
  }
}
__device__ __forceinline__ void vg_drain(uint32_t bar, uint32_t parity, long long limit_ns) {
  const unsigned long long t0 = global_ns();
  while (!mbar_try(bar, parity) && (long long)(global_ns() - t0) < limit_ns) {
  }
}
__device__ __forceinline__ float vg_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 32 bytes, a full sector, at once
__device__ __forceinline__ void vg_store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
template <bool F16>
__device__ __forceinline__ uint32_t vg_pack2(float a, float b) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
  }
}
// NC columns of a row from `col` on, those below N, in the element type of the operands (or float32)
template <class E, int NC>
__device__ __forceinline__ void vg_store_row(E* dst, int col, int N, const float* v) {
  if (col + NC <= N && ((uintptr_t)(dst + col) & 31) == 0) {
#pragma unroll
    for (int q = 0; q < NC; q += 32 / sizeof(E)) {
      if constexpr (sizeof(E) == 4) {
        vg_store32(dst + col + q, (const uint32_t*)(v + q));
      } else {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = vg_pack2<std::is_same_v<E, __half>>(v[q + 2 * i], v[q + 2 * i + 1]);
        vg_store32(dst + col + q, w);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (col + i < N) dst[col + i] = from_f<E>(v[i]);
  }
}

// OUT: element type of VG_OUT's result
// SEGS: the logits' reduction runs in segments whose sums are added in registers
template <int BN, bool AMN, bool BMN, int EPI, bool F16, bool SEGS, class OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kVgThreads, 1)
    k_vocab_gemm(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const VgArgs g) {
  constexpr int STAGES = vg_stages(BN), ACCS = BN == 512 ? 1 : 2;
  constexpr uint32_t A_BYTES = 128 * 64 * 2, B_BYTES = BN / 2 * 64 * 2;
  extern __shared__ unsigned char dsm[];
  __shared__ __align__(8) uint64_t bars[2 * STAGES + 4];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ float4 s_bias[EPI == VG_OUT ? 1 : kVgEpi][8];   // 32 columns' bias of each epilogue warp
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(dsm) + 1023u) & ~1023u, sA = base, sB = base + STAGES * A_BYTES;
  const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES]);
  const uint32_t acc_full = smem_u32(&bars[2 * STAGES]), acc_empty = smem_u32(&bars[2 * STAGES + 2]);
  volatile int* abort = &s_abort;
  uint32_t rank;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full + 8 * s, 1);
      mbar_init(acc_empty + 8 * s, 2 * kVgEpi);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&ma) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&mb) : "memory");
  }
  if (warp == kVgEpi + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"((uint32_t)(ACCS * BN))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  vg_meet();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  const int rows = *g.rows;
  const int M = g.M < 0 ? rows : g.M, K = g.K < 0 ? rows : g.K;
  const int tm = (M + 255) / 256, tn = (g.N + BN - 1) / BN;
  const int kb = (K + 63) / 64;
  const int seg = g.seg > 0 ? g.seg : max(1, (kb + g.splits - 1) / g.splits);   // 64-blocks of a segment
  const int nseg = (kb + seg - 1) / seg;
  // (the host has made sure that the items fit 32 bits)
  const unsigned items = (unsigned)tm * tn * g.splits, w0 = blockIdx.x >> 1, dw = gridDim.x >> 1;
  const auto tile_m = [&](unsigned w) { return (int)(w % (unsigned)tm); };
  const auto tile_n = [&](unsigned w) { return (int)(w / (unsigned)tm % (unsigned)tn); };
  const auto tile_s = [&](unsigned w) { return (int)(w / ((unsigned)tm * (unsigned)tn)); };
  // segments of part s of the reduction
  const auto first_seg = [&](int s) { return (int)((unsigned)(nseg * s) / (unsigned)g.splits); };

  if (warp == kVgEpi) {
    if (lane == 0) {
      unsigned it = 0;
      bool ok = true;
      for (unsigned w = w0; ok && w < items; w += dw) {
        const int m0 = tile_m(w) * 256 + (int)rank * 128, n0 = tile_n(w) * BN, sp = tile_s(w);
        const int bm = g.b_mn + n0 + (int)rank * (BN < 256 ? BN / 2 : 128);
        const int s1 = first_seg(sp + 1);
        for (int s = first_seg(sp); ok && s < s1; ++s) {
          const int k0 = s * seg, k1 = min(kb, k0 + seg);
          for (int p = 0; ok && p < g.nprod; ++p) {
            const int za = g.pa[p], zb = g.pb[p];
            for (int k = k0; k < k1; ++k, ++it) {
              const int st = it % STAGES;
              if (!vg_wait(empty0 + 8 * st, (it / STAGES & 1u) ^ 1u, g.spin_ns, abort, g.status)) {
                ok = false;
                break;
              }
              const uint32_t bar = vg_first(full0 + 8 * st), a = sA + st * A_BYTES, b = sB + st * B_BYTES;
              if (rank == 0) mbar_expect_tx(full0 + 8 * st, 2 * (A_BYTES + B_BYTES));
              const int ak = 64 * k, bk = g.b_k + 64 * k;
              if (AMN) {
#pragma unroll
                for (int q = 0; q < 2; ++q) vg_load(a + q * 8192, &ma, m0 + 64 * q, ak, za, bar);
              } else {
                vg_load(a, &ma, ak, m0, za, bar);
              }
              // of each 256 columns a CTA holds 128
              if (BMN) {
#pragma unroll
                for (int q = 0; q < BN / 128; ++q) vg_load(b + q * 8192, &mb, bm + q / 2 * 256 + q % 2 * 64, bk, zb, bar);
              } else {
                static_assert(BMN || BN <= 256, "one box");
                vg_load(b, &mb, bk, bm, zb, bar);
              }
            }
          }
        }
      }
      if (!ok && rank == 0)   // the pair's copies in flight: those of the last STAGES rounds
        for (unsigned j = it > STAGES ? it - STAGES : 0; j < it; ++j)
          vg_drain(full0 + 8 * (j % STAGES), j / STAGES & 1u, g.spin_ns);
    }
  } else if (warp == kVgEpi + 1) {
    if (lane == 0 && rank == 0) {
      // as for a single CTA, with M = 256 and the element types
      constexpr int MN = BN == 512 ? 256 : BN;
      constexpr uint32_t bf16 = umma_idesc_bf16(MN, AMN, BMN) + ((uint32_t)(128 >> 4) << 24);
      constexpr uint32_t idesc = F16 ? bf16 & ~((1u << 7) | (1u << 10)) : bf16;
      constexpr uint64_t astep = AMN ? (2048 >> 4) : (32 >> 4), bstep = BMN ? (2048 >> 4) : (32 >> 4);
      unsigned it = 0, acc = 0;
      bool ok = true;
      for (unsigned w = w0; ok && w < items; w += dw) {
        const int sp = tile_s(w), s1 = first_seg(sp + 1);
        for (int s = first_seg(sp); ok && s < s1; ++s, ++acc) {
          const int n = (min(kb, (s + 1) * seg) - s * seg) * g.nprod;
          const uint32_t d = tmem + (acc % ACCS) * BN;
          if (!(ok = vg_wait(acc_empty + 8 * (acc % ACCS), (acc / ACCS & 1u) ^ 1u, g.spin_ns, abort, g.status))) break;
          tc_fence_after();
          for (int j = 0; j < n; ++j, ++it) {
            const int st = it % STAGES;
            if (!(ok = vg_wait(full0 + 8 * st, it / STAGES & 1u, g.spin_ns, abort, g.status))) break;
            tc_fence_after();
            const uint64_t ad = umma_desc_sw128(sA + st * A_BYTES, AMN), bd = umma_desc_sw128(sB + st * B_BYTES, BMN);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              vg_mma(d, ad + astep * kk, bd + bstep * kk, idesc, j > 0 || kk > 0);
              if (BN == 512) vg_mma(d + 256, ad + astep * kk, bd + (16384 >> 4) + bstep * kk, idesc, j > 0 || kk > 0);
            }
            vg_commit(empty0 + 8 * st);
          }
          if (ok) vg_commit(acc_full + 8 * (acc % ACCS));
        }
      }
      if (!ok && it > 0) vg_drain(empty0 + 8 * ((it - 1) % STAGES), (it - 1) / STAGES & 1u, g.spin_ns);
    }
  } else {
    // ---- epilogue: row 32 (warp % 4) + lane of the tile, columns of half warp / 4
    const int half = warp >> 2, q = warp & 3;
    constexpr int HC = BN / 2;
    const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16) + half * HC;
    unsigned acc = 0;
    float whole[SEGS ? HC : 1];
    bool ok = true;
    for (unsigned w = w0; ok && w < items; w += dw) {
      const int m0 = tile_m(w) * 256 + (int)rank * 128, ct = tile_n(w), n0 = ct * BN + half * HC;
      const int sp = tile_s(w);
      const int s0 = first_seg(sp), s1 = first_seg(sp + 1);
      const int m = m0 + q * 32 + lane;
      // the next target's column, its place in the row's list, and the target behind it
      unsigned next = ~0u, after = ~0u;
      int pos = 0;
      const int* list = nullptr;
      if (EPI == VG_STATS && m < M) {
        list = g.idx + (long long)m * g.kept;
        if (!g.tab) {
          unsigned l[kVgFew];
#pragma unroll
          for (int k = 0; k < kVgFew; ++k) l[k] = k < g.kept ? (unsigned)list[k] : ~0u;
#pragma unroll
          for (int k = kVgFew - 1; k >= 0; --k) {
            if (l[k] >= (unsigned)n0) {
              after = next;
              next = l[k];
            } else {
              ++pos;
            }
          }
        } else {
          const unsigned t = g.tab[(2 * ct + half) * g.part_ld + m];
          pos = t >> 8;
          if ((t & 255) != 255) {
            next = n0 + (t & 255);
            if (pos + 1 < g.kept) after = list[pos + 1];
          }
        }
      }
      // a part without segments still writes its zeros
      for (int s = s0; ok && (s < s1 || s == s0); ++s) {
        const bool have = s < s1;
        const uint32_t t = lane_base + (acc % ACCS) * BN;
        if (have) {
          ok = vg_wait(acc_full + 8 * (acc % ACCS), acc / ACCS & 1u, g.spin_ns, abort, g.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
        }
        if constexpr (EPI != VG_OUT) {
          // VG_STATS: columns there are; VG_GRAD: columns of G
          const int limit = EPI == VG_STATS ? g.N : (int)g.g_ld;
          const bool in = m < M;
          const float lse = EPI == VG_GRAD && in ? g.lse[m] : 0.f, coef = EPI == VG_GRAD && in ? g.coef[m] : 0.f;
          float top = -INFINITY, sum = 0.f;
          // 32 columns of the row
          const auto chunk = [&](int n, float* v) {
            f2 w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pair(v[2 * i], v[2 * i + 1]);
            if (g.bias) {
              const float b = n + lane < g.N ? (g.bias_code == DELREC_F32 ? ((const float*)g.bias)[g.b_mn + n + lane]
                                               : F16 ? to_f(((const __half*)g.bias)[g.b_mn + n + lane])
                                                     : to_f(((const __nv_bfloat16*)g.bias)[g.b_mn + n + lane]))
                                             : 0.f;
              __syncwarp();
              ((float*)s_bias[warp])[lane] = b;
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 b4 = s_bias[warp][i];
                w[2 * i] = add2(w[2 * i], pair(b4.x, b4.y));
                w[2 * i + 1] = add2(w[2 * i + 1], pair(b4.z, b4.w));
              }
            }
            const f2 scale = pair(g.scale, g.scale);
            if constexpr (EPI == VG_STATS) {
#pragma unroll
              for (int i = 0; i < 16; ++i) split(w[i], v[2 * i], v[2 * i + 1]);
              if (n + 32 > g.N) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = n + i < g.N ? v[i] : -INFINITY;
              }
              unsigned at32;
              while ((at32 = next - (unsigned)n) < 32u) {
                float u[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) u[i] = at32 & 16 ? v[i + 16] : v[i];
#pragma unroll
                for (int o = 8; o; o >>= 1)
#pragma unroll
                  for (int i = 0; i < o; ++i) u[i] = at32 & o ? u[i + o] : u[i];
                g.z[(long long)m * g.kept + pos] = u[0];
                ++pos;
                next = after;
                after = pos + 1 < g.kept ? list[pos + 1] : ~0u;
              }
              __syncwarp();
              float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
              for (int i = 4; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], v[i]);
              const float mx = fmaxf(top, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * g.scale);
              const float at = mx == -INFINITY ? 0.f : mx;
              const f2 low = pair(-at, -at);
              f2 s2[2] = {pair(sum * vg_exp2(top - at), 0.f), pair(0.f, 0.f)};
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float a, b;
                split(fma2(pair(v[2 * i], v[2 * i + 1]), scale, low), a, b);
                s2[i & 1] = add2(s2[i & 1], pair(vg_exp2(a), vg_exp2(b)));
              }
              float s4[4];
              split(s2[0], s4[0], s4[1]);
              split(s2[1], s4[2], s4[3]);
              sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
              top = mx;
            } else {
              const f2 low = pair(-lse, -lse), c2 = pair(coef, coef);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float a, b;
                split(fma2(w[i], scale, low), a, b);
                split(mul2(pair(vg_exp2(a), vg_exp2(b)), c2), v[2 * i], v[2 * i + 1]);
              }
              if (n + 32 > g.N) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = n + i < g.N ? v[i] : 0.f;
              }
              if (m0 + q * 32 + 32 > M) {   // the last rows' tile
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = in ? v[i] : 0.f;
              }
              using E = std::conditional_t<F16, __half, __nv_bfloat16>;
              E* dst = (E*)g.G + (long long)m * g.g_ld + n;   // (a row's pitch is a multiple of 256)
              for (int pc = 0;; ++pc) {
                uint32_t h[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) h[i] = vg_pack2<F16>(v[2 * i], v[2 * i + 1]);
                vg_store32(dst, h);
                vg_store32(dst + 16, h + 8);
                if (pc + 1 == g.pieces) break;
                dst += g.g_piece;
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] -= to_f(from_f<E>(v[i]));   // what the piece leaves
              }
              __syncwarp();
            }
          };
          if constexpr (SEGS) {
#pragma unroll
            for (int c = 0; c < HC; c += 32)
              if (n0 + c < limit) {
                float v[32];
                tmem_ld32(t + c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) whole[c + i] = s == s0 ? v[i] : whole[c + i] + v[i];
              }
            if (s + 1 == s1) {
#pragma unroll
              for (int c = 0; c < HC; c += 32)
                if (n0 + c < limit) chunk(n0 + c, whole + c);
            }
          } else {
#pragma unroll 1
            for (int c = 0; c < HC && n0 + c < limit; c += 32) {
              float v[32];
              tmem_ld32(t + c, v);
              chunk(n0 + c, v);
            }
          }
          if (EPI == VG_STATS && in && s + 1 == s1) g.part[(2 * ct + half) * g.part_ld + m] = make_float2(top, sum);
        } else {
          const bool in = m < M;
          const float inv = g.out ? *g.inv : 1.f;
          const bool add = s > s0 || (!g.out && g.accumulate);
#pragma unroll 1
          for (int c = 0; c < HC; c += 32) {
            const int n = n0 + c;
            if (n >= g.N) break;
            float v[32];
            if (have) {
              tmem_ld32(t + c, v);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
            }
            if (!in) {
            } else if (g.out) {
              OUT* dst = (OUT*)g.out + (g.out0 + m) * g.out_ld;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= inv;
              if (add) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (n + i < g.N) v[i] += to_f(dst[n + i]);
              }
              vg_store_row<OUT, 32>(dst, n, g.N, v);
            } else {
              float* dst = g.plane + sp * g.plane_split + (long long)m * g.plane_ld;
              if (add) {
                if (n + 32 <= g.N && ((uintptr_t)(dst + n) & 15) == 0) {
#pragma unroll
                  for (int i = 0; i < 32; i += 4) {
                    const float4 o = *(const float4*)(dst + n + i);
                    v[i] += o.x; v[i + 1] += o.y; v[i + 2] += o.z; v[i + 3] += o.w;
                  }
                } else {
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (n + i < g.N) v[i] += dst[n + i];
                }
              }
              vg_store_row<float, 32>(dst, n, g.N, v);
            }
            __syncwarp();
          }
        }
        if (have) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) vg_arrive(vg_first(acc_empty + 8 * (acc % ACCS)));
          ++acc;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  vg_meet();
  if (warp == kVgEpi + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(ACCS * BN)) : "memory");
  }
}

}  // namespace delrec
