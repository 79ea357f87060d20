// Tensor-core products of the vocabulary losses (tcgen05 + TMA + tensor memory), fused with what
// follows them:
//
//   logits      z = x W^T (rows x vocabulary), never stored.  VG_STATS: each row's maximum and sum of
//               exponentials over the tile's columns.  VG_GRAD: c_m softmax(z)_mv in the operands'
//               type, from the row's log-sum-exp, for one piece of the vocabulary.
//   dW = G^T x  and  dx += G W  for that piece (VG_OUT).
//
// Persistent: one CTA per SM walks 128 x BN output tiles.  One thread streams operand tiles with TMA into
// a ring of shared-memory stages, one issues tcgen05.mma (M=128, N=BN, K=16) into one of two
// accumulators in tensor memory, eight warps read the other one back, so the epilogue of a tile runs
// under the next tile's products.  fp32 operands are three bf16 pieces each (an exact split) and six piece
// products, smallest first; 16-bit operands are taken as they are.  The tensor core's accumulator
// truncates, so long fp32 reductions run in segments whose sums are added outside it.
//
// The number of rows is read from the device (rows that do not count are packed away before).
// Every wait is bounded: on expiry the CTA records ST_TIMEOUT, drains its copies and returns.
#pragma once

#include "seq_common.cuh"
#include "tc_ptx.cuh"

namespace delrec {

enum { VG_STATS = 0, VG_GRAD = 1, VG_OUT = 2 };
constexpr int kVgThreads = 320;       // warps 0..7 epilogue, 8 TMA, 9 MMA
constexpr int kVgMaxProd = 6;
constexpr int kVgTimeout = 1 << 3;    // ST_TIMEOUT of the status word

struct VgArgs {
  const int* rows;              // device: rows that count
  int M, K;                     // output rows and reduction length; -1: *rows
  int N;                        // output columns
  int nprod, pa[kVgMaxProd], pb[kVgMaxProd];
  int a_mn, b_mn, a_k, b_k;     // where the operands start
  int splits, seg;              // reduction in `splits` parts of whole segments of `seg` 64-blocks (0: one per part)
  int* status;
  long long spin_ns;
  // VG_STATS: part[2 * column tile + half][row] = {max, sum}, in units of log2
  float2* part;
  long long part_ld;
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

constexpr int vg_stages(int BN) { return BN == 256 ? 4 : 6; }
constexpr size_t vg_smem(int BN) { return (size_t)vg_stages(BN) * (128 * 64 + BN * 64) * 2 + 1024; }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"((unsigned long long)map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void vg_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
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
template <int BN, bool AMN, bool BMN, int EPI, bool F16, class OUT>
__global__ void __launch_bounds__(kVgThreads, 1)
    k_vocab_gemm(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const VgArgs g) {
  constexpr int STAGES = vg_stages(BN);
  constexpr uint32_t A_BYTES = 128 * 64 * 2, B_BYTES = BN * 64 * 2;
  extern __shared__ unsigned char dsm[];
  __shared__ __align__(8) uint64_t bars[2 * STAGES + 4];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(dsm) + 1023u) & ~1023u, sA = base, sB = base + STAGES * A_BYTES;
  const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES]);
  const uint32_t acc_full = smem_u32(&bars[2 * STAGES]), acc_empty = smem_u32(&bars[2 * STAGES + 2]);
  volatile int* abort = &s_abort;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full + 8 * s, 1);
      mbar_init(acc_empty + 8 * s, 8);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&ma) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((unsigned long long)&mb) : "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"((uint32_t)(2 * BN))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  const int rows = *g.rows;
  const int M = g.M < 0 ? rows : g.M, K = g.K < 0 ? rows : g.K;
  const int tm = (M + 127) / 128, tn = (g.N + BN - 1) / BN;
  const int kb = (K + 63) / 64;
  const int seg = g.seg > 0 ? g.seg : max(1, (kb + g.splits - 1) / g.splits);   // 64-blocks of a segment
  const int nseg = (kb + seg - 1) / seg;
  const long long items = (long long)tm * tn * g.splits;
  // segments of part s of the reduction
  const auto first_seg = [&](int s) { return (int)((long long)nseg * s / g.splits); };

  if (warp == 8) {
    if (lane == 0) {
      unsigned it = 0;
      bool ok = true;
      for (long long w = blockIdx.x; ok && w < items; w += gridDim.x) {
        const int m0 = (int)(w % tm) * 128, n0 = (int)(w / tm % tn) * BN, sp = (int)(w / ((long long)tm * tn));
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
              const uint32_t bar = full0 + 8 * st, a = sA + st * A_BYTES, b = sB + st * B_BYTES;
              mbar_expect_tx(bar, A_BYTES + B_BYTES);
              const int ak = g.a_k + 64 * k, bk = g.b_k + 64 * k, am = g.a_mn + m0, bm = g.b_mn + n0;
              if (AMN) {
#pragma unroll
                for (int q = 0; q < 2; ++q) tma_load_3d(a + q * 8192, &ma, am + 64 * q, ak, za, bar);
              } else {
                tma_load_3d(a, &ma, ak, am, za, bar);
              }
              if (BMN) {
#pragma unroll
                for (int q = 0; q < BN / 64; ++q) tma_load_3d(b + q * 8192, &mb, bm + 64 * q, bk, zb, bar);
              } else {
                tma_load_3d(b, &mb, bk, bm, zb, bar);
              }
            }
          }
        }
      }
      if (!ok)   // the copies in flight: those of the last STAGES rounds
        for (unsigned j = it > STAGES ? it - STAGES : 0; j < it; ++j)
          vg_drain(full0 + 8 * (j % STAGES), j / STAGES & 1u, g.spin_ns);
    }
  } else if (warp == 9) {
    if (lane == 0) {
      constexpr uint32_t idesc = F16 ? umma_idesc_bf16(BN, AMN, BMN) & ~((1u << 7) | (1u << 10)) : umma_idesc_bf16(BN, AMN, BMN);
      constexpr uint64_t astep = AMN ? (2048 >> 4) : (32 >> 4), bstep = BMN ? (2048 >> 4) : (32 >> 4);
      unsigned it = 0, acc = 0;
      bool ok = true;
      for (long long w = blockIdx.x; ok && w < items; w += gridDim.x) {
        const int sp = (int)(w / ((long long)tm * tn)), s1 = first_seg(sp + 1);
        for (int s = first_seg(sp); ok && s < s1; ++s, ++acc) {
          const int n = (min(kb, (s + 1) * seg) - s * seg) * g.nprod;
          const uint32_t d = tmem + (acc & 1) * BN;
          if (!(ok = vg_wait(acc_empty + 8 * (acc & 1), (acc / 2 & 1u) ^ 1u, g.spin_ns, abort, g.status))) break;
          tc_fence_after();
          for (int j = 0; j < n; ++j, ++it) {
            const int st = it % STAGES;
            if (!(ok = vg_wait(full0 + 8 * st, it / STAGES & 1u, g.spin_ns, abort, g.status))) break;
            tc_fence_after();
            const uint64_t ad = umma_desc_sw128(sA + st * A_BYTES, AMN), bd = umma_desc_sw128(sB + st * B_BYTES, BMN);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) umma_bf16(d, ad + astep * kk, bd + bstep * kk, idesc, j > 0 || kk > 0);
            umma_commit(empty0 + 8 * st);
          }
          if (ok) umma_commit(acc_full + 8 * (acc & 1));
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
    bool ok = true;
    for (long long w = blockIdx.x; ok && w < items; w += gridDim.x) {
      const int m0 = (int)(w % tm) * 128, ct = (int)(w / tm % tn), n0 = ct * BN + half * HC;
      const int sp = (int)(w / ((long long)tm * tn));
      const int s0 = first_seg(sp), s1 = first_seg(sp + 1);
      const int m = m0 + q * 32 + lane;
      // a part without segments still writes its zeros
      for (int s = s0; ok && (s < s1 || s == s0); ++s) {
        const bool have = s < s1;
        const uint32_t t = lane_base + (acc & 1) * BN;
        if (have) {
          ok = vg_wait(acc_full + 8 * (acc & 1), acc / 2 & 1u, g.spin_ns, abort, g.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
        }
        if constexpr (EPI == VG_STATS) {
          float top = -INFINITY, sum = 0.f;
#pragma unroll 1
          for (int c = 0; c < HC; c += 32) {
            const int n = n0 + c;
            if (n >= g.N) break;
            float v[32];
            tmem_ld32(t + c, v);
            if (g.bias) {
              const float b = n + lane < g.N ? (g.bias_code == DELREC_F32 ? ((const float*)g.bias)[g.b_mn + n + lane]
                                               : F16 ? to_f(((const __half*)g.bias)[g.b_mn + n + lane])
                                                     : to_f(((const __nv_bfloat16*)g.bias)[g.b_mn + n + lane]))
                                             : 0.f;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, b, i);
            }
            if (n + 32 > g.N) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = n + i < g.N ? v[i] : -INFINITY;
            }
            float mx = v[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) mx = fmaxf(mx, v[i]);
            mx = fmaxf(top, mx * g.scale);
            const float at = mx == -INFINITY ? 0.f : mx;
            float s4[4] = {sum * vg_exp2(top - at), 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 32; ++i) s4[i & 3] += vg_exp2(fmaf(v[i], g.scale, -at));
            sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
            top = mx;
          }
          if (m < M) g.part[(2 * ct + half) * g.part_ld + m] = make_float2(top, sum);
        } else if constexpr (EPI == VG_GRAD) {
          const bool in = m < M;
          const float lse = in ? g.lse[m] : 0.f, coef = in ? g.coef[m] : 0.f;
#pragma unroll 1
          for (int c = 0; c < HC; c += 32) {
            const int n = n0 + c;
            if (n >= g.g_ld) break;
            float v[32];
            tmem_ld32(t + c, v);
            if (g.bias) {
              const float b = n + lane < g.N ? (g.bias_code == DELREC_F32 ? ((const float*)g.bias)[g.b_mn + n + lane]
                                               : F16 ? to_f(((const __half*)g.bias)[g.b_mn + n + lane])
                                                     : to_f(((const __nv_bfloat16*)g.bias)[g.b_mn + n + lane]))
                                             : 0.f;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, b, i);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = coef * vg_exp2(fmaf(v[i], g.scale, -lse));
            if (n + 32 > g.N) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = n + i < g.N ? v[i] : 0.f;
            }
            if (!in) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
            }
            using E = std::conditional_t<F16, __half, __nv_bfloat16>;
            E* dst = (E*)g.G + (long long)m * g.g_ld;
            for (int pc = 0; pc < g.pieces; ++pc) {
              vg_store_row<E, 32>(dst + pc * g.g_piece, n, (int)g.g_ld, v);
              if (pc + 1 < g.pieces) {   // what the piece leaves
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] -= to_f(from_f<E>(v[i]));
              }
            }
            __syncwarp();
          }
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
          if (lane == 0) vg_arrive(acc_empty + 8 * (acc & 1));
          ++acc;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * BN)) : "memory");
  }
}

}  // namespace delrec
