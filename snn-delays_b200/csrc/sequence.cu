// extern "C" entry points of the block norms and the 8-bit checkpoints: argument checks, kernel
// variants and launch shapes.  No allocation happens here.
#include <algorithm>

#include "block_norm.cuh"
#include "checkpoint8.cuh"
#include "seq_common.cuh"

namespace delrec {

// --------------------------------------------------------------------------------
// block norm
// --------------------------------------------------------------------------------
static constexpr int kNormMax = 16384;

static int check_block(const delrec_block* s) {
  if (!s || s->T < 1 || s->B < 1 || s->N < 1) return DELREC_ERR_ARG;
  if (s->dtype < DELREC_F32 || s->dtype > DELREC_F16 || s->gate < GATE_NONE || s->gate > GATE_SILU)
    return DELREC_ERR_ARG;
  if (!(s->eps > 0.f)) return DELREC_ERR_ARG;
  if (s->N > kNormMax || (long long)s->T * s->B > 0x7fffffffLL - 4 * kSeqSMs * 16) return DELREC_ERR_UNSUPPORTED;
  for (long long st : {s->x_t, s->x_b, s->y_t, s->y_b, s->u_t, s->u_b, s->o_t, s->o_b, s->n_t, s->n_b, s->gx_t,
                       s->gx_b, s->gn_t, s->gn_b, s->dx_t, s->dx_b, s->dy_t, s->dy_b, s->du_t, s->du_b})
    if (st < -0x7fffffffLL || st > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  return DELREC_OK;
}

// May every row of these tensors be read and written V elements at a time?  Do their rows lie
// one pitch apart?
struct NormAlign {
  int esz, B;
  bool ok[2];   // 8 and 16 bytes
  long long pitch = -1;   // -1: none seen, 0: not shared
  NormAlign(int esz_, int N, int B_) : esz(esz_), B(B_) {
    ok[0] = (size_t)N * esz % 8 == 0;
    ok[1] = (size_t)N * esz % 16 == 0;
  }
  void add(const void* ptr, long long st, long long sb) {
    if (!ptr) return;
    const unsigned long long m = (unsigned long long)(uintptr_t)ptr | (unsigned long long)(st * esz) |
                                 (unsigned long long)(sb * esz);
    if (m & 7) ok[0] = false;
    if (m & 15) ok[1] = false;
    if (st != B * sb || (pitch >= 0 && sb != pitch)) pitch = 0;
    else pitch = sb;
  }
  int flat(long long rows) const { return pitch > 0 && rows * pitch < 0x7fffffffLL ? (int)pitch : 0; }
};

static NormShape norm_shape(int N, int V, int esz, int most_threads) {
  NormShape s{};
  s.V = V;
  const int vecs = (N + V - 1) / V;
  // 16 bytes of each tensor to a thread where that leaves a warp: what a row costs besides its
  // channels (addresses, two sums) is some 130 operations a thread (fp16 N=700 in 8-byte
  // vectors, one of them 61 us, two 47 us); more costs blocks per SM (fp32 N=512 forward, 16 bytes
  // 111 us, 32 bytes 125 us).  N <= 16384: at most 32 channels.
  s.IT = 1;
  while (s.IT * V * esz < 16 && vecs > 32 * s.IT) s.IT *= 2;
  while ((vecs + s.IT - 1) / s.IT > most_threads) s.IT *= 2;
  s.threads = ((vecs + s.IT - 1) / s.IT + 31) / 32 * 32;
  return s;
}
static int norm_most_blocks(const delrec_block* s) {
  return (int)std::min<long long>((long long)s->T * s->B, (long long)kSeqSMs * 16);
}
static size_t norm_bwd_ws(const delrec_block* s) { return (size_t)norm_most_blocks(s) * 2 * s->N * sizeof(float); }

static int norm_width(const NormAlign& al) { return al.ok[1] ? 16 / al.esz : (al.ok[0] ? 8 / al.esz : 1); }

static NormArgs norm_args(const delrec_block* s) {
  NormArgs a{};
  a.T = s->T; a.B = s->B; a.N = s->N; a.wide = s->lengths_wide; a.eps = s->eps;
  a.x_t = (int)s->x_t; a.x_b = (int)s->x_b; a.y_t = (int)s->y_t; a.y_b = (int)s->y_b; a.u_t = (int)s->u_t; a.u_b = (int)s->u_b;
  a.o_t = (int)s->o_t; a.o_b = (int)s->o_b; a.n_t = (int)s->n_t; a.n_b = (int)s->n_b;
  a.gx_t = (int)s->gx_t; a.gx_b = (int)s->gx_b; a.gn_t = (int)s->gn_t; a.gn_b = (int)s->gn_b;
  a.dx_t = (int)s->dx_t; a.dx_b = (int)s->dx_b; a.dy_t = (int)s->dy_t; a.dy_b = (int)s->dy_b; a.du_t = (int)s->du_t; a.du_b = (int)s->du_b;
  return a;
}

// --------------------------------------------------------------------------------
// 8-bit checkpoints
// --------------------------------------------------------------------------------
template <class T, int V, bool PACK>
static int q8_launch(Q8Args a, cudaStream_t st) {
  constexpr int L = 32 / V, most = 512;
  a.gpr = (a.N + kQGroup - 1) / kQGroup;
  a.span = a.gpr * L;
  a.rpb = std::max(1, most / a.span);
  const int threads = std::min(most, a.span * a.rpb);
  const long long blocks = (a.rows + a.rpb - 1) / a.rpb;
  void (*kern)(Q8Args) = PACK ? k_pack8<T, V> : k_unpack8<T, V>;
  int per_sm = 1;   // as many blocks as fit at once
  if (blocks > kSeqSMs) SQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, 0));
  const int grid = (int)std::min<long long>(blocks, (long long)kSeqSMs * std::max(per_sm, 1));
  kern<<<grid, threads, 0, st>>>(a);
  SQ_LAUNCHED();
  return DELREC_OK;
}
// 16 bytes of x a thread where every row is so aligned, 8 of a 16-bit type, else one value
template <class T, bool PACK>
static int q8_run(const Q8Args& a, const void* x, cudaStream_t st) {
  constexpr int V16 = 16 / sizeof(T), V8 = 8 / sizeof(T);
  const auto fits = [&](int V) {
    return a.N % V == 0 && (uintptr_t)x % (V * sizeof(T)) == 0 && (uintptr_t)a.q % V == 0;
  };
  if (fits(V16)) return q8_launch<T, V16, PACK>(a, st);
  if (fits(V8)) return q8_launch<T, V8, PACK>(a, st);
  return q8_launch<T, 1, PACK>(a, st);
}

}  // namespace delrec

using namespace delrec;

extern "C" {

int delrec_block_norm_forward(const delrec_block* s, const void* x, const void* y, const void* u, const float* w,
                              const float* scale, const float* next_w, const void* lengths, void* out, void* n,
                              float* ry, float* rx, void* stream) {
  const int rc = check_block(s);
  if (rc) return rc;
  if (!x || (y && !out) || (!y && !n) || (y && s->gate != GATE_NONE && !u)) return DELREC_ERR_ARG;
  NormArgs a = norm_args(s);
  a.x = x; a.y = y; a.u = u; a.w = w; a.scale = scale; a.nw = next_w; a.lengths = lengths;
  a.out = out; a.n = n; a.ry = ry; a.rx = rx;
  const int gate = y ? s->gate : GATE_NONE;
  NormAlign al(s->dtype == DELREC_F32 ? 4 : 2, s->N, s->B);
  al.add(x, s->x_t, s->x_b);
  al.add(n, s->n_t, s->n_b);
  if (y) {
    al.add(y, s->y_t, s->y_b);
    al.add(out, s->o_t, s->o_b);
    if (gate != GATE_NONE) al.add(u, s->u_t, s->u_b);
  }
  NormShape sh = norm_shape(s->N, norm_width(al), al.esz, kNormThreads);
  a.kind = gate;
  a.pitch = al.flat((long long)s->T * s->B);
  return norm_run_forward(s->dtype, a, sh, norm_most_blocks(s), (cudaStream_t)stream);
}

size_t delrec_block_norm_backward_workspace(const delrec_block* s) { return check_block(s) ? 0 : norm_bwd_ws(s); }

int delrec_block_norm_backward(const delrec_block* s, const void* x, const void* y, const void* u, const float* w,
                               const float* scale, const float* next_w, const void* lengths, const float* ry,
                               const float* rx, const void* gx, const void* gn, void* dx, void* dy, void* du,
                               float* dw, float* dscale, float* dnext_w, void* ws, size_t wsb, void* stream) {
  const int rc = check_block(s);
  if (rc) return rc;
  if ((y && !ry) || (gn && (!rx || !x)) || (y && s->gate != GATE_NONE && !u)) return DELREC_ERR_ARG;
  const bool sums = dw || dscale || dnext_w;
  if (sums && (!ws || ((uintptr_t)ws & 255) != 0 || wsb < norm_bwd_ws(s))) return DELREC_ERR_WORKSPACE;
  NormArgs a = norm_args(s);
  a.x = x; a.y = y; a.u = u; a.w = w; a.scale = scale; a.nw = next_w; a.lengths = lengths;
  a.ry = const_cast<float*>(ry); a.rx = const_cast<float*>(rx);
  a.gx = gx; a.gn = gn; a.dx = dx; a.dy = dy; a.du = du; a.part = sums ? (float*)ws : nullptr;
  const int gate = y ? s->gate : GATE_NONE;
  NormAlign al(s->dtype == DELREC_F32 ? 4 : 2, s->N, s->B);
  if (gn) al.add(x, s->x_t, s->x_b);
  al.add(gx, s->gx_t, s->gx_b);
  al.add(gn, s->gn_t, s->gn_b);
  al.add(dx, s->dx_t, s->dx_b);
  if (y) {
    al.add(y, s->y_t, s->y_b);
    al.add(dy, s->dy_t, s->dy_b);
    if (gate != GATE_NONE) {
      al.add(u, s->u_t, s->u_b);
      al.add(du, s->du_t, s->du_b);
    }
  }
  NormShape sh = norm_shape(s->N, norm_width(al), al.esz, kNormThreads);
  a.kind = gate;
  a.pitch = al.flat((long long)s->T * s->B);
  const cudaStream_t st = (cudaStream_t)stream;
  const int r = norm_run_backward(s->dtype, a, sh, norm_most_blocks(s), st);
  if (r || !sums) return r;
  k_norm_dw<<<dim3((s->N + 31) / 32, dnext_w ? 2 : 1), 1024, 0, st>>>(s->N, sh.grid, (const float*)ws, w, scale, dw, dscale, dnext_w);
  SQ_LAUNCHED();
  return DELREC_OK;
}

int delrec_pack8(long long rows, int N, int dtype, const void* x, int8_t* q, uint8_t* e, void* stream) {
  if (rows < 0 || N < 1 || rows > (1LL << 62) / N || !x || !q || !e) return DELREC_ERR_ARG;
  if (rows == 0) return DELREC_OK;
  Q8Args a{};
  a.rows = rows; a.N = N; a.x = x; a.q = q; a.e = e;
  return by_dtype(dtype, [&](auto t) { return q8_run<decltype(t), true>(a, x, (cudaStream_t)stream); });
}

int delrec_unpack8(long long rows, int N, int dtype, const int8_t* q, const uint8_t* e, void* x, void* stream) {
  if (rows < 0 || N < 1 || rows > (1LL << 62) / N || !x || !q || !e) return DELREC_ERR_ARG;
  if (rows == 0) return DELREC_OK;
  Q8Args a{};
  a.rows = rows; a.N = N; a.out = x; a.q = const_cast<int8_t*>(q); a.e = const_cast<uint8_t*>(e);
  return by_dtype(dtype, [&](auto t) { return q8_run<decltype(t), false>(a, x, (cudaStream_t)stream); });
}

}  // extern "C"
