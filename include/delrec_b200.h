/*
 * delrec_b200: C-ABI of the B200-native delay-LIF hot path (DelRec).
 *
 * All pointers are device pointers, tensors are fp32, contiguous, time-major (T,B,N).
 * Weights follow the reference's convention W[i,o] (row = target neuron i, column =
 * source neuron o): rec[b,i] = sum_o W[i,o] * (delayed spike of o).
 * Every entry point launches on `stream` (a cudaStream_t; NULL = legacy default stream)
 * and returns DELREC_OK or an error code.  Scratch memory is passed in by the caller:
 * query its size with the matching *_workspace function.  Weight gradients, the
 * synaptic lag stack, the projections, the chunked reverse scan and the step-by-step
 * forward and reverse scans of axonal layers wider than 512 neurons run on the library's
 * own tcgen05 GEMM; the library calls no vendor math library.
 *
 * Reference interfaces replaced (paths are inside ZiyadBekrar/SNN-delays):
 *   delrec_build_mask             triton_kernels/delays.py:13-29, 48-63 (build_mask,
 *                                 build_syn_mask)
 *   delrec_axonal_forward         triton_kernels/recdel_base.py:136-182 (recdel_triton_forward,
 *                                 launching recdel_fwd_kernel :34-129)
 *   delrec_axonal_backward        recdel_base.py:288-342 (recdel_triton_backward: recdel_bwd_kernel
 *                                 :189-285 + host dW/db/dmask) and the dmask->dd/dp autograd
 *                                 of AxonalRecdelTriton.backward :402-439
 *   delrec_synaptic_forward       triton_kernels/synaptic_eventdriven.py:386-416 (EventDrivenSyn
 *                                 .forward launching _ed_scatter_compact_kernel :106-164)
 *   delrec_synaptic_backward      synaptic_eventdriven.py:419-471 (EventDrivenSyn.backward:
 *                                 _ed_bwd_kernel :323-364 + Cstack GEMMs + autograd dd/dp)
 *   delrec_hybrid_forward         triton_kernels/synaptic_hybrid.py:139-172 (HybridSynDelay.forward)
 *   delrec_hybrid_backward        synaptic_hybrid.py:175-211 (HybridSynDelay.backward incl.
 *                                 _hybrid_dd_kernel :83-113), with the (N,N) delay gradient
 *                                 already reduced onto the learned (N,) base the way the
 *                                 parametrization networks.py:823-829 does
 *   delrec_hybrid_delay_grad      synaptic_hybrid.py:116-126 (_delay_grad, closed-form dd)
 *   delrec_lif_forward/backward   the multi-step SpikingJelly LIFNode used between layers by
 *                                 the model zoo (networks.py:84-96), no recurrence
 *   delrec_dcls_forward/backward  networks.py:43-50 (dcls_module.forward: DCLS 0.1.1 Gaussian
 *                                 kernel construction + causal conv1d over time)
 *   delrec_linear_forward/backward  the torch.nn.Linear projections between the delay layers
 *                                 and the readout (networks.py:84-96, 140-181)
 */
#ifndef DELREC_B200_H
#define DELREC_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---------------------------------------------------------------- */
#define DELREC_OK 0
#define DELREC_ERR_ARG 1          /* invalid size / null pointer / bad enum            */
#define DELREC_ERR_CUDA 2         /* a CUDA launch or attribute call failed             */
#define DELREC_ERR_WORKSPACE 3    /* workspace too small or misaligned (256 B)          */
#define DELREC_ERR_UNSUPPORTED 4  /* shape outside the kernels' supported range          */

/* ---- delay kinds ------------------------------------------------------------------ */
#define DELREC_AXONAL 0           /* d (N,): one delay per source neuron                */
#define DELREC_SYNAPTIC 1         /* d (N,N): one delay per connection d[i,o]           */
#define DELREC_HYBRID 2           /* learned base (N,) + frozen integer offsets (N,N)   */

/* surrogate ids: identical to triton_kernels/surrogate.py:_SURR_ID */
#define DELREC_SURR_TRIANGLE 0
#define DELREC_SURR_ATAN 1

/* LIF neuron, SpikingJelly LIFNode semantics with decay_input=False
 * (charge v*(1-1/tau)+a when v_reset is None or 0, else v-(v-v_reset)/tau+a; fire
 * u-v_th >= 0; hard reset to v_reset or soft reset by v_th; initial v = v_reset, or 0
 * for a soft reset). */
typedef struct delrec_lif {
  float tau;
  float v_threshold;
  float v_reset;        /* ignored when soft_reset != 0 */
  int32_t soft_reset;   /* 1: v_reset is None */
  int32_t detach_reset; /* 1: no gradient through the reset */
  int32_t surrogate;    /* DELREC_SURR_* */
  float gamma;          /* Triangle width */
  float alpha;          /* ATan slope */
} delrec_lif;

/* Shape and delay description of one recurrent delay layer. */
typedef struct delrec_layer {
  int32_t kind;         /* DELREC_AXONAL / DELREC_SYNAPTIC / DELREC_HYBRID */
  int32_t T, B, N;
  int32_t L;            /* ring length ceil(1 + max d + max s) + 1 (lags 1..L-1) */
  int32_t K;            /* hybrid: largest integer offset (offsets in [0, K]) */
  int32_t has_bias;     /* bias pointer is read */
  int32_t has_keep;     /* keep (B,N) dropout mask is read */
  float s_max;          /* largest triangle half-width (1 + sigma, or max over s) */
  float d_min;          /* smallest delay (hybrid: smallest learned base; may be negative) */
} delrec_layer;

/* Gradient outputs of a layer backward.  Any pointer may be NULL to skip it. */
typedef struct delrec_grads {
  float* dx;            /* (T,B,N) */
  float* dW;            /* (N,N)   */
  float* dbias;         /* (N,)    */
  float* dd;            /* axonal (N,), synaptic (N,N), hybrid base (N,) */
  float* ds;            /* (N,) gradient w.r.t. the per-source half-width s (use_sig_p) */
} delrec_grads;

/* Triangle delay kernel h[r,l] = max(0, s_r' - |l - (1 + d[r])|) / s_r'^2 for l in [0,L),
 * rows r in [0,R); s_r' = s[r % s_period] (s_period = N for synaptic (N,N) delays whose
 * width is indexed by the source, = R for axonal).  out (R, L). */
int delrec_build_mask(int R, int L, const float* d, const float* s, int s_period,
                      float* out, void* stream);

/* ---- axonal layer ------------------------------------------------------------------ */
/* x (T,B,N), W (N,N), bias (N), d (N), s (N) half-widths, keep (B,N).
 * Outputs y (spikes) and u (pre-reset membrane), both (T,B,N). */
size_t delrec_axonal_forward_workspace(const delrec_layer* layer);
int delrec_axonal_forward(const delrec_layer* layer, const delrec_lif* lif,
                          const float* x, const float* W, const float* bias,
                          const float* d, const float* s, const float* keep,
                          float* y, float* u, void* workspace, size_t workspace_bytes,
                          void* stream);
/* gy (T,B,N) upstream gradient of the spikes; u, y from the forward. */
size_t delrec_axonal_backward_workspace(const delrec_layer* layer);
int delrec_axonal_backward(const delrec_layer* layer, const delrec_lif* lif,
                           const float* gy, const float* u, const float* y,
                           const float* W, const float* d, const float* s,
                           const float* keep, const delrec_grads* grads,
                           void* workspace, size_t workspace_bytes, void* stream);

/* Hard-tap forms of the axonal layer: AxonalRecdelTriton with ste_mode 1 / 2 or approx
 * (triton_kernels/recdel_base.py:350-445, recdel_bwd_kernel APPROX branch :215-278).
 * Their forwards are delrec_axonal_forward at half-width s = 1 with the hard taps written
 * as a delay: the single tap at lag l (lag = clamp(round(d) + 1, 1, .)) is d = l - 1 and
 * the two-tap interpolation (1 - f) at l, f at l + 1 (l = floor(1 + d)) is d = l - 1 + f,
 * i.e. max(d, 0).  Backwards:
 *   DELREC_HARD_STE     the soft triangle's backward over (d, s) -- gfut, dx, dd, ds,
 *                       dbias -- except dW, which correlates gr with the hard forward's z
 *                       (taps of d_hard at half-width 1);
 *   DELREC_HARD_APPROX  the backward of the single-tap forward: d = the hard delays
 *                       (l - 1), s all 1 and the layer's L sized for them; dd is the
 *                       straight-through sum_{t,b} gz[t,b,n] (y[t-l-1,b,n] - y[t-l,b,n]);
 *                       grads->ds must be NULL, d_hard is not read. */
#define DELREC_HARD_STE 1
#define DELREC_HARD_APPROX 2
size_t delrec_axonal_backward_hard_workspace(const delrec_layer* layer);
int delrec_axonal_backward_hard(const delrec_layer* layer, const delrec_lif* lif, int mode,
                                const float* gy, const float* u, const float* y,
                                const float* W, const float* d, const float* s,
                                const float* d_hard, const float* keep,
                                const delrec_grads* grads, void* workspace,
                                size_t workspace_bytes, void* stream);

/* ---- the library's own tensor-core GEMM (tcgen05, bf16 pieces, fp32 accumulate) ------
 * No reference counterpart as an interface: it is the contraction engine behind the
 * weight gradients, the lag-correlation stack and the projections (which the reference
 * runs as torch matmuls / cuBLAS), exposed so it can be tested on its own.
 * D (M,N) = [D +] sum_p A[prod_a[p]] . B[prod_b[p]]^T over K.  layout bit 0: A pieces
 * are stored (K,M) instead of (M,K) (MN-major); bit 1: B pieces (K,N) instead of (N,K).
 * Pieces are bf16, 16-byte aligned, row strides lda / ldb multiples of 8 elements; D fp32
 * row stride ldd.  ksplit > 1 splits the reduction (partials in the workspace, summed in
 * a fixed order); block_n = 64, 128 or 256 output columns per tile. */
size_t delrec_tc_gemm_workspace(int M, int N, int ksplit);
int delrec_tc_gemm(int M, int N, int K, int layout, int a_pieces, const void* const* A, long long lda,
                   int b_pieces, const void* const* B, long long ldb, int nprod, const int* prod_a,
                   const int* prod_b, int ksplit, int block_n, float* D, long long ldd, int accumulate,
                   void* workspace, size_t workspace_bytes, void* stream);

/* Same as delrec_axonal_forward but allocation-free: no reference counterpart.  It is for
 * callers that cannot call cudaMalloc while the layer runs (all device memory handed to
 * their own allocator, no device-wide synchronisation allowed in the loop, or a plugin
 * host that forbids allocation after start-up).  Its scratch is a fixed 8 MiB device
 * array inside the library, held by every GPU that loads the library until the process
 * exits.  Limits: N <= 1024 neurons (wider layers get DELREC_ERR_WORKSPACE); every width
 * runs the per-sample scan, whose spike history lives in shared memory, so very long
 * rings (at N = 1024, L above about 1000) get DELREC_ERR_UNSUPPORTED.  The first call on
 * a device looks the array up (cudaGetSymbolAddress), so make that first call before any
 * stream capture.  All calls share the array: calls that overlap on the GPU (other
 * streams, other threads) race on it.  Every byte it reads is written earlier in the
 * same call, so nothing carries over between calls. */
int delrec_axonal_forward_noalloc(const delrec_layer* layer, const delrec_lif* lif,
                                  const float* x, const float* W, const float* bias,
                                  const float* d, const float* s, const float* keep,
                                  float* y, float* u, void* stream);

/* ---- synaptic layer ---------------------------------------------------------------- */
/* d (N,N) per connection, s (N) per source. */
size_t delrec_synaptic_forward_workspace(const delrec_layer* layer);
int delrec_synaptic_forward(const delrec_layer* layer, const delrec_lif* lif,
                            const float* x, const float* W, const float* bias,
                            const float* d, const float* s, const float* keep,
                            float* y, float* u, void* workspace, size_t workspace_bytes,
                            void* stream);
size_t delrec_synaptic_backward_workspace(const delrec_layer* layer);
int delrec_synaptic_backward(const delrec_layer* layer, const delrec_lif* lif,
                             const float* gy, const float* u, const float* y,
                             const float* W, const float* d, const float* s,
                             const float* keep, const delrec_grads* grads,
                             void* workspace, size_t workspace_bytes, void* stream);

/* ---- hybrid layer ------------------------------------------------------------------ */
/* base (N,) learned per source, offsets (N,N) frozen integers in [0,K] (fp32, as the
 * reference buffer); effective delay d[i,o] = base[o] + offsets[i,o].  s (N). */
size_t delrec_hybrid_forward_workspace(const delrec_layer* layer);
int delrec_hybrid_forward(const delrec_layer* layer, const delrec_lif* lif,
                          const float* x, const float* W, const float* bias,
                          const float* base, const float* offsets, const float* s,
                          const float* keep, float* y, float* u,
                          void* workspace, size_t workspace_bytes, void* stream);
/* The backward factors each synapse's delay into base + offset and supports base tap
 * windows that reach at most one lag below lag 1 (layer->d_min, s_max); a wider window
 * returns DELREC_ERR_UNSUPPORTED -- run such a layer through delrec_synaptic_* on the
 * materialised delay d[i,o] = base[o] + offsets[i,o] (the Python Function does). */
size_t delrec_hybrid_backward_workspace(const delrec_layer* layer);
int delrec_hybrid_backward(const delrec_layer* layer, const delrec_lif* lif,
                           const float* gy, const float* u, const float* y,
                           const float* W, const float* base, const float* offsets,
                           const float* s, const float* keep, const delrec_grads* grads,
                           void* workspace, size_t workspace_bytes, void* stream);

/* Closed-form per-synapse delay gradient of the hybrid/synaptic triangle kernel:
 * dd[i,o] = W[i,o] * sum_{l=1}^{LM-1} C[i,o,l] * g(l - 1 - d[i,o]),
 * g(a) = sign(a)/s^2 where |a| <= s, else 0  (s = 1 + sigma).  C (N,N,LM). */
int delrec_hybrid_delay_grad(int N, int LM, const float* C, const float* W,
                             const float* d, float sigma, float* dd, void* stream);

/* ---- plain multi-step LIF (no recurrence) ------------------------------------------ */
int delrec_lif_forward(int T, int M, const delrec_lif* lif, const float* x,
                       float* y, float* u, void* stream);
int delrec_lif_backward(int T, int M, const delrec_lif* lif, const float* gy,
                        const float* u, float* dx, void* stream);

/* ---- DCLS feedforward delay (Gaussian-interpolated positions, causal conv) ---------- */
/* x (T,B,Cin); weight (Cout, Cin/groups); P, SIG (Cout, Cin/groups); kernel width K;
 * left zero padding lpad (= K-1 for the causal length-preserving layer).  out (T,B,Cout).
 * The constructed dense kernel is written to ker (Cout, Cin/groups, K). */
int delrec_dcls_forward(int T, int B, int Cin, int Cout, int groups, int K, int lpad,
                        const float* x, const float* weight, const float* P,
                        const float* SIG, const float* bias, float* ker, float* out,
                        void* stream);
/* Gradients w.r.t. x, weight, P, SIG, bias (any may be NULL).  gout (T,B,Cout). */
size_t delrec_dcls_backward_workspace(int T, int B, int Cin, int Cout, int groups, int K);
int delrec_dcls_backward(int T, int B, int Cin, int Cout, int groups, int K, int lpad,
                         const float* x, const float* weight, const float* P,
                         const float* SIG, const float* gout, float* dx, float* dweight,
                         float* dP, float* dSIG, float* dbias,
                         void* workspace, size_t workspace_bytes, void* stream);

/* ---- feedforward projection ------------------------------------------------------- */
/* out (M,N) = x (M,K) . W^T + bias, W (N,K) as torch.nn.Linear, bias (N) or NULL.
 * Runs on bf16 tensor cores with fp32 accuracy: each fp32 operand is split exactly into
 * three bf16 pieces and the piece products with i + j <= 2 are summed with fp32
 * accumulation.  x_binary = 1 promises x in {0, 1} (spike trains: three products instead
 * of six); a violated promise sets the status word.  The GEMMs run on the library's
 * tcgen05 GEMM (partials on a slice of the workspace). */
size_t delrec_linear_forward_workspace(int M, int K, int N, int x_binary);
int delrec_linear_forward(int M, int K, int N, const float* x, const float* W, const float* bias,
                          int x_binary, float* out, void* workspace, size_t workspace_bytes,
                          void* stream);
/* gout (M,N); dx (M,K), dW (N,K), dbias (N): any may be NULL (x may be NULL when dW and
 * dbias are, W when dx is). */
size_t delrec_linear_backward_workspace(int M, int K, int N, int x_binary);
int delrec_linear_backward(int M, int K, int N, const float* x, const float* W, const float* gout,
                           int x_binary, float* dx, float* dW, float* dbias, void* workspace,
                           size_t workspace_bytes, void* stream);

/* ---- readout + time sum of the loss ----------------------------------------------- */
/* The model zoo's readout Linear (networks.py:140-181) followed by the SSC / PS-MNIST
 * loss's sum over time (utils.py:188-200, calc_loss_SSC), fused: out (B,C) =
 * sum_t (y_t W^T + bias) = ysum W^T + T bias with ysum (B,N) = sum_t y_t written too; the
 * (T,B,C) readout is never formed.  y (T,B,N), W (C,N) as torch.nn.Linear, bias (C) or
 * NULL.  Backward with g (B,C) = dloss/dout: dy (T,B,N) = g W for every t, dW (C,N) =
 * g^T ysum, dbias (C) = T sum_b g (any output may be NULL).  fp32, fixed summation order. */
int delrec_readout_sum_forward(int T, int B, int N, int C, const float* y, const float* W,
                               const float* bias, float* ysum, float* out, void* stream);
int delrec_readout_sum_backward(int T, int B, int N, int C, const float* ysum, const float* W,
                                const float* g, float* dy, float* dW, float* dbias, void* stream);

/* Sets *count (device) to the number of entries of x[0..n) that are neither 0 nor 1;
 * asynchronous on the stream, x 16-byte aligned.  The projections' spike-input test
 * (x_binary above); no counterpart in the reference, whose projections are fp32 GEMMs. */
int delrec_count_nonbinary(const float* x, size_t n, unsigned int* count, void* stream);

/* ---- sequence operators ------------------------------------------------------------ */
/* Gated linear recurrence, norms around a block, 8-bit activation checkpoints: no
 * counterpart in the reference.  Tensors are fp32, bf16 or fp16 (dtype), time-major
 * (T,B,N) with element strides for T and B and contiguous channels; states, weights,
 * statistics and their gradients are fp32.  lengths (B), int32 or int64
 * (lengths_wide != 0), NULL for full rows: positions t >= lengths[b] are not read, their
 * outputs and gradients are written as 0.  Outputs do not overlap inputs unless stated.
 * Pointers and strides are aligned to their element type; wider accesses are chosen where
 * they allow them. */
#define DELREC_F32 0
#define DELREC_BF16 1
#define DELREC_F16 2
#define DELREC_GATE_NONE 0
#define DELREC_GATE_SIGMOID 1
#define DELREC_GATE_SILU 2

typedef struct delrec_scan {
  int32_t T, B, N;
  int32_t G;             /* gates per position; N = G * D, gate g serves channels gD .. gD+D-1 */
  int32_t dtype;
  int32_t decay_input;   /* 1: z enters as (1 - a) z, 0: as z */
  int32_t lengths_wide;
  int32_t reserved;
  int64_t z_t, z_b, f_t, f_b;       /* strides of z (T,B,N) and f (T,B,G) */
  int64_t h_t, h_b;                 /* of h */
  int64_t gh_t, gh_b;               /* of the gradient of h */
  int64_t dz_t, dz_b, df_t, df_b;   /* of dz and df */
} delrec_scan;

/* h_t = sigmoid(f_t) h_{t-1} + c_t z_t from h0 (B,N) (NULL: 0); resets (T,B) bytes or NULL:
 * nonzero drops h_{t-1} at that step.  Writes h, hT (B,N) (the state after the last
 * position; NULL to skip) and, for the backward, states (ceil(T/16), B, N): the state before
 * every 16th step (NULL to skip).  qz, ez, qf, ef, odd (all or none, G = N): also writes z
 * and f in 8 bits (delrec_pack8's form), and odd (ceil(T/16), B, ceil(N/32)): nonzero where a
 * code of those 16 steps and 32 channels may stand for an infinity or NaN.  T, and B times the
 * tiles of at most 32 channels of a row, are at most 2^30, B N below 2^31. */
int delrec_gated_scan_forward(const delrec_scan* scan, const void* z, const void* f, const float* h0,
                              const void* lengths, const uint8_t* resets, void* h, float* hT, float* states,
                              int8_t* qz, uint8_t* ez, int8_t* qf, uint8_t* ef, uint8_t* odd, void* stream);
/* Gradients from gh (NULL: 0) and ghT (NULL: 0): dz, df, dh0, any NULL to skip.  With qz,
 * ez, qf, ef, odd (all or none, G = N), z and f are what those stand for.  h_{t-1} is recomputed
 * from states. */
size_t delrec_gated_scan_backward_workspace(const delrec_scan* scan);
int delrec_gated_scan_backward(const delrec_scan* scan, const void* z, const void* f, const int8_t* qz,
                               const uint8_t* ez, const int8_t* qf, const uint8_t* ef, const uint8_t* odd,
                               const void* lengths, const uint8_t* resets, const float* states, const void* gh, const float* ghT,
                               void* dz, void* df, float* dh0, void* workspace, size_t workspace_bytes,
                               void* stream);
/* One step (T is 1): h (B,N) and next (B,N) from z, f and state (B,N) (NULL: 0); next may be
 * state itself.  active (B) bytes or NULL: a row with 0 keeps its state and writes h = 0. */
int delrec_gated_step(const delrec_scan* scan, const void* z, const void* f, const float* state,
                      const uint8_t* active, void* h, float* next, void* stream);

typedef struct delrec_block {
  int32_t T, B, N;
  int32_t dtype;
  int32_t gate;          /* DELREC_GATE_* */
  int32_t lengths_wide;
  float eps;             /* > 0 */
  int32_t reserved;
  int64_t x_t, x_b, y_t, y_b, u_t, u_b;         /* strides of x, y, u */
  int64_t o_t, o_b, n_t, n_b;                   /* of the outputs x' and n */
  int64_t gx_t, gx_b, gn_t, gn_b;               /* of their gradients */
  int64_t dx_t, dx_b, dy_t, dy_b, du_t, du_b;   /* of dx, dy, du */
} delrec_block;

/* out = x + scale * act(u) * (y / rms(y) * w) and n = out / rms(out) * next_w, rms(v) =
 * sqrt(mean v^2 + eps) over the channels.  y NULL: n is x's norm, out is not written.  n
 * NULL: no next norm.  w, scale, next_w (N), NULL: ones.  ry, rx (T,B), NULL to skip: the
 * 1/rms of y and of out, kept for the backward.  N <= 16384. */
int delrec_block_norm_forward(const delrec_block* block, const void* x, const void* y, const void* u,
                              const float* w, const float* scale, const float* next_w, const void* lengths,
                              void* out, void* n, float* ry, float* rx, void* stream);
/* Gradients from gx (of out) and gn (of n), either NULL: 0.  Outputs NULL to skip. */
size_t delrec_block_norm_backward_workspace(const delrec_block* block);
int delrec_block_norm_backward(const delrec_block* block, const void* x, const void* y, const void* u,
                               const float* w, const float* scale, const float* next_w, const void* lengths,
                               const float* ry, const float* rx, const void* gx, const void* gn, void* dx,
                               void* dy, void* du, float* dw, float* dscale, float* dnext_w, void* workspace,
                               size_t workspace_bytes, void* stream);

/* 8-bit form of x (rows, N), contiguous: q (rows, N) and e (rows, ceil(N/32)).  Channels
 * go in groups of 32; x is q * 2^(e-127), the scale the smallest power of two >= 2^-126
 * with max |x| <= 126 * scale over the group's finite values, q = x / scale rounded to
 * nearest even (at the scale 2^122 at most 63 in magnitude); q = 127 is +inf, -127 -inf,
 * -128 NaN.  Restored to fp16 it saturates at fp16's largest value. */
int delrec_pack8(long long rows, int N, int dtype, const void* x, int8_t* q, uint8_t* e, void* stream);
int delrec_unpack8(long long rows, int N, int dtype, const int8_t* q, const uint8_t* e, void* x, void* stream);
/* delrec_linear_forward that also writes x (M,K) in 8 bits, q and e as delrec_pack8, from the
 * same read (same workspace).  A real x's piece products are summed smallest first, which
 * is a little more exact; for x_binary = 1 out has delrec_linear_forward's bits. */
int delrec_linear_forward8(int M, int K, int N, const float* x, const float* W, const float* bias, int x_binary,
                           float* out, int8_t* q, uint8_t* e, void* workspace, size_t workspace_bytes,
                           void* stream);
/* delrec_linear_backward with x in 8 bits: its values have 7 significant bits, so one bf16
 * piece carries each exactly and dW takes three piece products. */
size_t delrec_linear_backward8_workspace(int M, int K, int N);
int delrec_linear_backward8(int M, int K, int N, const int8_t* q, const uint8_t* e, const float* W,
                            const float* gout, float* dx, float* dW, float* dbias, void* workspace,
                            size_t workspace_bytes, void* stream);

/* ---- short causal convolution ----------------------------------------------------------- */
/* p_t = bias + sum_j w[:,j] x_{t-K+1+j}, y = act(p), one filter of K <= 8 taps per channel.  x, y,
 * their gradients and the states are of one element type; w (N,K) and bias (N) float32.  Strides
 * are in elements; channels are contiguous. */
typedef struct delrec_conv {
  int32_t T, B, N, K;
  int32_t dtype;
  int32_t act;           /* 0 none, 1 silu */
  int32_t lengths_kind;  /* lengths (B): 0 int32, 1 int64, 2 one byte (a row has T steps or none) */
  int32_t reserved;
  int64_t x_t, x_b, y_t, y_b, gy_t, gy_b, dx_t, dx_b;
} delrec_conv;

/* state (K-1,B,N), NULL: zeros: the inputs before the first step, oldest first; next (K-1,B,N), NULL
 * to skip: the last K-1 of each sequence.  With T = 1, next may be state.  bias NULL: 0.  lengths,
 * resets NULL: whole sequences.  Rows past a length are not read, their y is 0. */
int delrec_short_conv_forward(const delrec_conv* conv, const void* x, const float* w, const float* bias,
                              const void* state, const void* lengths, const uint8_t* resets, void* y, void* next,
                              void* stream);
/* Gradients from gy (of y) and gs (of next), either NULL: 0.  Outputs NULL to skip; the workspace
 * serves dw (N,K) and db (N). */
size_t delrec_short_conv_backward_workspace(const delrec_conv* conv);
int delrec_short_conv_backward(const delrec_conv* conv, const void* x, const float* w, const float* bias,
                               const void* state, const void* lengths, const uint8_t* resets, const void* gy,
                               const void* gs, void* dx, void* ds, float* dw, float* db, void* workspace,
                               size_t workspace_bytes, void* stream);

/* ---- selective state space scan ------------------------------------------------------------ */
/* delta = softplus(dt + dt_bias) (softplus = 0: without softplus), h_t[n,s] = exp(delta A[n,s])
 * h_{t-1}[n,s] + delta B_t[g,s] x_t[n], y_t[n] = (sum_s C_t[g,s] h_t[n,s] + D[n] x_t[n]) silu(gate_t[n]);
 * group g serves N / G channels; S <= 128.  x, dt, gate, y (T,B,N) and Bm, Cm (T,B,G,S) of one element
 * type; A (N,S), D, dt_bias (N), states (.., N,S) float32.  bm_*, cm_*: strides of T and B; (G,S) are
 * contiguous. */
typedef struct delrec_selective {
  int32_t T, B, N, S, G;
  int32_t dtype;
  int32_t softplus;
  int32_t lengths_wide;  /* lengths are int64 */
  int32_t ragged;        /* there are lengths (a hint: how time is cut; the same in every call of a pass) */
  int32_t no_bc;         /* backward: neither dB nor dC is wanted; their partial sums then take no workspace */
  int64_t x_t, x_b, dt_t, dt_b, u_t, u_b, y_t, y_b;             /* x, dt, gate, y */
  int64_t bm_t, bm_b, cm_t, cm_b;                               /* Bm, Cm */
  int64_t gy_t, gy_b, dx_t, dx_b, ddt_t, ddt_b, du_t, du_b;     /* gradients of y, x, dt, gate */
} delrec_selective;

/* D, gate, dt_bias, h0 (B,N,S), lengths, resets (T,B): NULL for none.  hT (B,N,S) the state after the
 * last step.  states (ceil(T/8),B,N,S), NULL without a backward pass: the state before every 8th.
 * 16-byte aligned where S % 4 == 0: hT, states, dh0.  Rows past a length are not read, their y is 0. */
size_t delrec_selective_forward_workspace(const delrec_selective* s);
int delrec_selective_forward(const delrec_selective* s, const void* x, const void* dt, const float* A, const void* Bm,
                             const void* Cm, const float* D, const void* gate, const float* dt_bias, const float* h0,
                             const void* lengths, const uint8_t* resets, void* y, float* hT, float* states,
                             void* workspace, size_t workspace_bytes, void* stream);
/* Gradients from gy (of y) and ghT (of hT), either NULL: 0.  Outputs NULL to skip; dB, dC (T,B,G,S)
 * contiguous. */
size_t delrec_selective_backward_workspace(const delrec_selective* s);
int delrec_selective_backward(const delrec_selective* s, const void* x, const void* dt, const float* A, const void* Bm,
                              const void* Cm, const float* D, const void* gate, const float* dt_bias,
                              const void* lengths, const uint8_t* resets, const float* states, const void* gy,
                              const float* ghT, void* dx, void* ddt, float* dA, void* dB, void* dC, float* dD,
                              void* dgate, float* ddt_bias, float* dh0, void* workspace, size_t workspace_bytes,
                              void* stream);
/* One time step (T = 1) of state (B,N,S) (NULL: 0) into next, which may be state.  active (B) bytes,
 * NULL: all; a row that is not keeps its state and gives y = 0.  y (B,N) contiguous. */
int delrec_selective_step(const delrec_selective* s, const void* x, const void* dt, const float* A, const void* Bm,
                          const void* Cm, const float* D, const void* gate, const float* dt_bias, const float* state,
                          const uint8_t* active, void* y, float* next, void* stream);

/* ---- losses of a projection onto a vocabulary ------------------------------------------------ */
/* Of z = x W^T + bias, which is never stored, over the T * B positions of x:
 *   cross entropy   loss_m = logsumexp(z_m) - z_m[index_m]
 *   distillation    loss_m = tau^2 sum_k p_k (log p_k - log q[index_mk]), p = softmax(logits_m / tau)
 *                   over the K kept entries, q = softmax(z_m / tau) over the vocabulary
 * x (T,B,D), W (V,D), bias (V) of one element type; W and bias contiguous.  A position does not count
 * (loss and gradient 0) at or past lengths[b], where index is ignore_index, or where its list keeps
 * nothing: an entry with a negative index or a logit of -inf is left out.  An index that is V or more
 * (or negative and not ignore_index) makes the loss NaN and sets a bit of the status word.  D <= 8192,
 * K <= 1024, T * B <= 2^24, V <= 2^30. */
typedef struct delrec_vocab {
  int32_t T, B, D, V, K;     /* K = 1 for the cross entropy */
  int32_t dtype;
  int32_t distill;
  int32_t reduction;         /* 0 none: out (T,B); 1 mean over the positions that count; 2 sum: out (1) */
  int32_t lengths_wide;      /* lengths are int64 */
  int32_t index_wide;        /* index is int64 */
  int32_t teacher_dtype;     /* of logits */
  int32_t w_aligned;         /* W is 16-byte aligned */
  float temperature;         /* tau, 1e-6 to 1e6; 1 for the cross entropy */
  int32_t split;             /* backward: the logits' gradient of a 16-bit type in two pieces of it, also past 512 positions */
  int64_t ignore_index;
  int64_t x_t, x_b;
} delrec_vocab;

/* keep: what the backward pass takes over (256-byte aligned, as the workspaces). */
size_t delrec_vocab_loss_keep(const delrec_vocab* s);
size_t delrec_vocab_loss_forward_workspace(const delrec_vocab* s);
int delrec_vocab_loss_forward(const delrec_vocab* s, const void* x, const void* w, const void* bias, const void* index,
                              const void* logits, const void* lengths, float* out, void* keep, size_t keep_bytes,
                              void* workspace, size_t workspace_bytes, void* stream);
/* Gradients from g (of out).  dx (T,B,D), dw (V,D), db (V) contiguous, NULL to skip. */
size_t delrec_vocab_loss_backward_workspace(const delrec_vocab* s);
int delrec_vocab_loss_backward(const delrec_vocab* s, const void* x, const void* w, const void* bias, const float* g,
                               const void* keep, size_t keep_bytes, void* dx, void* dw, void* db, void* workspace,
                               size_t workspace_bytes, void* stream);

/* ---- device status word ------------------------------------------------------------ */
/* Kernels record internal inconsistencies (an out-of-range lag or index that was
 * skipped) in a device status word instead of trapping.  Reading it synchronizes. */
int delrec_get_status(int* status_out);
int delrec_clear_status(void);
const char* delrec_version(void);
/* Number of kernels this library has launched in this process (host-side counter). */
unsigned long long delrec_launch_count(void);
/* Measurement hooks: while enabled, every reverse-scan launch (the backward's time loop)
 * is bracketed by CUDA events on its stream; delrec_scan_time synchronizes on them and
 * returns the summed milliseconds and the number of launches since enabling. */
int delrec_scan_timing(int enable);
int delrec_scan_time(double* total_ms, int* launches);
/* The same per part: 0 = every reverse scan (a chunked scan counts as one launch per
 * layer), 1 = the step launches of the chunked scans, 2 = their chunk GEMM launches. */
int delrec_scan_time_part(int part, double* total_ms, int* launches);
/* Reverse-scan variant of the layer backwards (process-wide).  0 (default): hybrid layers
 * whose shape allows it run the chunked scan -- the delayed-gradient contraction of every
 * synapse whose lag reaches past the current 8-step chunk as one tensor-core GEMM per
 * chunk, the short-lag synapses step by step in blocks that own whole samples; 1: the
 * step-by-step scans only; 2: the chunked scan with its steps split over source slices
 * that exchange gr through L2 every step (kept for comparison).  All give
 * the reference's gradients within the library's tolerance; the workspace size queries
 * cover either variant.  Replaces no reference call (the reference has one Triton
 * kernel per layer kind, triton_kernels/synaptic_eventdriven.py:323-364). */
int delrec_set_reverse_scan(int variant);
/* Measurement: the per-step latency floor of the reverse scans.  Runs T steps of their
 * exchange alone -- each block publishes its slice of gr to L2, meets its batch tile at an
 * arrival counter and restages the tile's gr into shared memory -- on the grid and tiling
 * the 64-sample scans use for `layer` (N <= 512, B > 32; otherwise
 * DELREC_ERR_UNSUPPORTED), with no LIF step and no synapse sums.  Time it with events on
 * `stream`.  No counterpart in the reference. */
size_t delrec_exchange_floor_workspace(const delrec_layer* layer);
int delrec_exchange_floor(const delrec_layer* layer, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DELREC_B200_H */
