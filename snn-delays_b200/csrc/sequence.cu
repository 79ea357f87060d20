// extern "C" entry points of the sequence operators: argument checks, kernel variants and
// launch shapes.  No allocation happens here.
#include <algorithm>

#include "block_norm.cuh"
#include "checkpoint8.cuh"
#include "gated_scan.cuh"
#include "seq_common.cuh"

namespace delrec {

static int seq_grid(size_t n, int threads, int per_sm) {
  const size_t g = (n + threads - 1) / threads;
  return (int)std::max<size_t>(1, std::min(g, (size_t)kSeqSMs * per_sm));
}

// calls fn(T()) with the element type
template <class F>
static int by_dtype(int dtype, F&& fn) {
  switch (dtype) {
    case DELREC_F32: return fn(float());
    case DELREC_BF16: return fn(__nv_bfloat16());
    case DELREC_F16: return fn(__half());
  }
  return DELREC_ERR_ARG;
}

// --------------------------------------------------------------------------------
// gated scan
// --------------------------------------------------------------------------------
static int check_scan(const delrec_scan* s) {
  if (!s || s->T < 1 || s->B < 1 || s->N < 1 || s->G < 1 || s->N % s->G != 0) return DELREC_ERR_ARG;
  if (s->dtype < DELREC_F32 || s->dtype > DELREC_F16) return DELREC_ERR_ARG;
  if (s->T > (1 << 30)) return DELREC_ERR_UNSUPPORTED;
  return DELREC_OK;
}

struct ScanShape {
  int P, csize;
  unsigned grid;
};

static int scan_shape(const delrec_scan* s, ScanArgs* p, ScanShape* sh) {
  p->T = s->T; p->B = s->B; p->N = s->N; p->G = s->G; p->D = s->N / s->G;
  p->decay_input = s->decay_input; p->wide = s->lengths_wide;
  if (p->D > 32) {
    p->tph = (p->D + 31) / 32;
    p->cpt = 32;
    p->tiles = p->G * p->tph;
  } else {
    p->tph = 0;
    p->cpt = 32 / p->D * p->D;
    p->tiles = (p->N + p->cpt - 1) / p->cpt;
  }
  const long long items = (long long)p->B * p->tiles;
  const int segs = (p->T + kSeg - 1) / kSeg;
  sh->P = segs >= kScanWarps ? kScanWarps : 1;
  // few rows: the blocks of a cluster share one row's time
  int c = 1;
  while (c < kScanCluster && items * c < 2 * kSeqSMs && sh->P * c * 2 <= segs) c *= 2;
  sh->csize = c;
  if (items * c > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  sh->grid = (unsigned)(items * c);
  return DELREC_OK;
}

static int scan_launch(void (*kern)(ScanArgs, int), ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(sh.grid);
  cfg.blockDim = dim3(sh.P * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = sh.csize;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = sh.csize > 1 ? 1 : 0;
  SQ_CUDA(cudaLaunchKernelEx(&cfg, kern, p, (int)sh.csize));
  SQ_LAUNCHED();
  return DELREC_OK;
}

template <class T, int P, bool POS>
static int scan_fwd_p(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
  return scan_launch(p.qz ? k_scan_fwd<T, P, POS, true> : k_scan_fwd<T, P, POS, false>, p, sh, st);
}
template <class T, int P, bool POS>
static int scan_bwd_p(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
  return scan_launch(p.qz ? k_scan_bwd<T, P, POS, true> : k_scan_bwd<T, P, POS, false>, p, sh, st);
}

// --------------------------------------------------------------------------------
// block norm
// --------------------------------------------------------------------------------
static constexpr int kNormMax = 16384;

static int check_block(const delrec_block* s) {
  if (!s || s->T < 1 || s->B < 1 || s->N < 1) return DELREC_ERR_ARG;
  if (s->dtype < DELREC_F32 || s->dtype > DELREC_F16 || s->gate < GATE_NONE || s->gate > GATE_SILU)
    return DELREC_ERR_ARG;
  if (!(s->eps > 0.f)) return DELREC_ERR_ARG;
  if (s->N > kNormMax) return DELREC_ERR_UNSUPPORTED;
  return DELREC_OK;
}

// may every row of these tensors be read and written V elements at a time?
struct NormAlign {
  int esz;
  bool ok[2];   // 8 and 16 bytes
  explicit NormAlign(int esz_, int N) : esz(esz_) {
    ok[0] = (size_t)N * esz % 8 == 0;
    ok[1] = (size_t)N * esz % 16 == 0;
  }
  void add(const void* ptr, long long st, long long sb) {
    if (!ptr) return;
    const unsigned long long m = (unsigned long long)(uintptr_t)ptr | (unsigned long long)(st * esz) |
                                 (unsigned long long)(sb * esz);
    if (m & 7) ok[0] = false;
    if (m & 15) ok[1] = false;
  }
};

struct NormShape {
  int V, IT, threads, grid;
};
static NormShape norm_shape(int N, long long rows, int V, int most_threads) {
  NormShape s;
  s.V = V;
  const int vecs = (N + V - 1) / V;
  s.IT = 1;
  while ((vecs + s.IT - 1) / s.IT > most_threads) s.IT *= 2;   // N <= 16384: at most 32 elements a thread
  s.threads = ((vecs + s.IT - 1) / s.IT + 31) / 32 * 32;
  const int per_sm = std::max(1, std::min(16, 1024 / s.threads));
  s.grid = (int)std::min<long long>(rows, (long long)kSeqSMs * per_sm);
  return s;
}

using NormKernel = void (*)(NormArgs);
template <class T, int V, bool BWD, bool GATE, int IT = 1>
static NormKernel norm_kernel(int it) {
  if constexpr (V * IT <= 32) {
    if (it == IT) return BWD ? k_norm_bwd<T, V, IT, GATE> : k_norm_fwd<T, V, IT, GATE>;
    return norm_kernel<T, V, BWD, GATE, 2 * IT>(it);
  }
  return nullptr;
}
template <class T, int V, bool BWD>
static int norm_launch(NormArgs a, int gate, const NormShape& s, cudaStream_t st) {
  NormKernel k = gate == GATE_NONE ? norm_kernel<T, V, BWD, false>(s.IT) : norm_kernel<T, V, BWD, true>(s.IT);
  if (!k) return DELREC_ERR_UNSUPPORTED;
  a.kind = gate;
  k<<<s.grid, s.threads, 0, st>>>(a);
  SQ_LAUNCHED();
  return DELREC_OK;
}
// the widest access the tensors allow, 16 bytes at most
template <class T, bool BWD>
static int norm_run(const NormArgs& a, int gate, const NormShape& s, cudaStream_t st) {
  constexpr int V16 = 16 / sizeof(T), V8 = 8 / sizeof(T);
  if (s.V == V16) return norm_launch<T, V16, BWD>(a, gate, s, st);
  if (s.V == V8) return norm_launch<T, V8, BWD>(a, gate, s, st);
  return norm_launch<T, 1, BWD>(a, gate, s, st);
}
static int norm_width(const NormAlign& al) { return al.ok[1] ? 16 / al.esz : (al.ok[0] ? 8 / al.esz : 1); }
static int norm_most_blocks(const delrec_block* s) {
  return (int)std::min<long long>((long long)s->T * s->B, (long long)kSeqSMs * 16);
}
static size_t norm_bwd_ws(const delrec_block* s) { return (size_t)norm_most_blocks(s) * 2 * s->N * sizeof(float); }

static NormArgs norm_args(const delrec_block* s) {
  NormArgs a{};
  a.T = s->T; a.B = s->B; a.N = s->N; a.wide = s->lengths_wide; a.eps = s->eps;
  a.x_t = s->x_t; a.x_b = s->x_b; a.y_t = s->y_t; a.y_b = s->y_b; a.u_t = s->u_t; a.u_b = s->u_b;
  a.o_t = s->o_t; a.o_b = s->o_b; a.n_t = s->n_t; a.n_b = s->n_b;
  a.gx_t = s->gx_t; a.gx_b = s->gx_b; a.gn_t = s->gn_t; a.gn_b = s->gn_b;
  a.dx_t = s->dx_t; a.dx_b = s->dx_b; a.dy_t = s->dy_t; a.dy_b = s->dy_b; a.du_t = s->du_t; a.du_b = s->du_b;
  return a;
}

}  // namespace delrec

using namespace delrec;

extern "C" {

int delrec_gated_scan_forward(const delrec_scan* s, const void* z, const void* f, const float* h0,
                              const void* lengths, const uint8_t* resets, void* h, float* hT, float* states,
                              int8_t* qz, uint8_t* ez, int8_t* qf, uint8_t* ef, void* stream) {
  int rc = check_scan(s);
  if (rc) return rc;
  if (!z || !f || !h) return DELREC_ERR_ARG;
  const bool pack = qz || ez || qf || ef;
  if (pack && (!(qz && ez && qf && ef) || s->G != s->N)) return DELREC_ERR_ARG;
  ScanArgs p{};
  ScanShape sh;
  if ((rc = scan_shape(s, &p, &sh))) return rc;
  p.z = z; p.f = f; p.h0 = h0; p.lengths = lengths; p.resets = resets; p.h = h; p.hT = hT; p.states = states;
  p.qz = qz; p.ez = ez; p.qf = qf; p.ef = ef;
  p.z_t = s->z_t; p.z_b = s->z_b; p.f_t = s->f_t; p.f_b = s->f_b; p.h_t = s->h_t; p.h_b = s->h_b;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pos = lengths || resets;
  return by_dtype(s->dtype, [&](auto t) {
    using T = decltype(t);
    if (sh.P == 1) return pos ? scan_fwd_p<T, 1, true>(p, sh, st) : scan_fwd_p<T, 1, false>(p, sh, st);
    return pos ? scan_fwd_p<T, kScanWarps, true>(p, sh, st) : scan_fwd_p<T, kScanWarps, false>(p, sh, st);
  });
}

size_t delrec_gated_scan_backward_workspace(const delrec_scan* s) {
  if (check_scan(s)) return 0;
  const int D = s->N / s->G;
  return D > 32 ? (size_t)s->T * s->B * s->G * ((D + 31) / 32) * sizeof(float) : 0;
}

int delrec_gated_scan_backward(const delrec_scan* s, const void* z, const void* f, const int8_t* qz,
                               const uint8_t* ez, const int8_t* qf, const uint8_t* ef, const void* lengths,
                               const uint8_t* resets, const float* states, const void* gh, const float* ghT,
                               void* dz, void* df, float* dh0, void* ws, size_t wsb, void* stream) {
  int rc = check_scan(s);
  if (rc) return rc;
  if (!states || (!qz != !ez) || (!qf != !ef) || (!qz && !z) || (!qf && !f) || (qf && !qz)) return DELREC_ERR_ARG;
  ScanArgs p{};
  ScanShape sh;
  if ((rc = scan_shape(s, &p, &sh))) return rc;
  const size_t need = df ? delrec_gated_scan_backward_workspace(s) : 0;
  if (need && (!ws || ((uintptr_t)ws & 255) != 0 || wsb < need)) return DELREC_ERR_WORKSPACE;
  p.z = z; p.f = f; p.lengths = lengths; p.resets = resets; p.states = const_cast<float*>(states);
  p.qz = const_cast<int8_t*>(qz); p.ez = const_cast<uint8_t*>(ez);
  p.qf = const_cast<int8_t*>(qf); p.ef = const_cast<uint8_t*>(ef);
  p.gh = gh; p.ghT = ghT; p.dz = dz; p.df = df; p.dh0 = dh0; p.part = (float*)ws;
  p.z_t = s->z_t; p.z_b = s->z_b; p.f_t = s->f_t; p.f_b = s->f_b; p.gh_t = s->gh_t; p.gh_b = s->gh_b;
  p.dz_t = s->dz_t; p.dz_b = s->dz_b; p.df_t = s->df_t; p.df_b = s->df_b;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pos = lengths || resets;
  return by_dtype(s->dtype, [&](auto t) {
    using T = decltype(t);
    int r;
    if (sh.P == 1) r = pos ? scan_bwd_p<T, 1, true>(p, sh, st) : scan_bwd_p<T, 1, false>(p, sh, st);
    else r = pos ? scan_bwd_p<T, kScanWarps, true>(p, sh, st) : scan_bwd_p<T, kScanWarps, false>(p, sh, st);
    if (r) return r;
    if (df && p.tph) {
      k_scan_df_sum<T><<<seq_grid((size_t)p.T * p.B * p.G, 256, 8), 256, 0, st>>>(p);
      SQ_LAUNCHED();
    }
    return (int)DELREC_OK;
  });
}

int delrec_gated_step(const delrec_scan* s, const void* z, const void* f, const float* state,
                      const uint8_t* active, void* h, float* next, void* stream) {
  const int rc = check_scan(s);
  if (rc) return rc;
  if (s->T != 1 || !z || !f || !h || !next) return DELREC_ERR_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  return by_dtype(s->dtype, [&](auto t) {
    using T = decltype(t);
    k_gated_step<T><<<seq_grid((size_t)s->B * s->N, 128, 16), 128, 0, st>>>(
        s->B, s->N, s->N / s->G, s->decay_input, (const T*)z, s->z_b, (const T*)f, s->f_b, state, active, (T*)h,
        next);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  });
}

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
  NormAlign al(s->dtype == DELREC_F32 ? 4 : 2, s->N);
  al.add(x, s->x_t, s->x_b);
  al.add(n, s->n_t, s->n_b);
  if (y) {
    al.add(y, s->y_t, s->y_b);
    al.add(out, s->o_t, s->o_b);
    if (gate != GATE_NONE) al.add(u, s->u_t, s->u_b);
  }
  const NormShape sh = norm_shape(s->N, (long long)s->T * s->B, norm_width(al), kNormThreads);
  return by_dtype(s->dtype, [&](auto t) {
    return norm_run<decltype(t), false>(a, gate, sh, (cudaStream_t)stream);
  });
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
  NormAlign al(s->dtype == DELREC_F32 ? 4 : 2, s->N);
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
  const NormShape sh = norm_shape(s->N, (long long)s->T * s->B, norm_width(al), kNormThreads);
  const cudaStream_t st = (cudaStream_t)stream;
  const int r = by_dtype(s->dtype, [&](auto t) { return norm_run<decltype(t), true>(a, gate, sh, st); });
  if (r || !sums) return r;
  k_norm_dw<<<(s->N + 31) / 32, 256, 0, st>>>(s->N, sh.grid, (const float*)ws, w, scale, dw, dscale, dnext_w);
  SQ_LAUNCHED();
  return DELREC_OK;
}

int delrec_pack8(long long rows, int N, int dtype, const void* x, int8_t* q, uint8_t* e, void* stream) {
  if (rows < 0 || N < 1 || rows > (1LL << 62) / N || !x || !q || !e) return DELREC_ERR_ARG;
  if (rows == 0) return DELREC_OK;
  const int gpr = (N + kQGroup - 1) / kQGroup;
  const long long groups = rows * gpr;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_pack8<T><<<seq_grid((size_t)groups, 8, 16), 256, 0, (cudaStream_t)stream>>>(groups, gpr, N, (const T*)x, q, e);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  });
}

int delrec_unpack8(long long rows, int N, int dtype, const int8_t* q, const uint8_t* e, void* x, void* stream) {
  if (rows < 0 || N < 1 || rows > (1LL << 62) / N || !x || !q || !e) return DELREC_ERR_ARG;
  if (rows == 0) return DELREC_OK;
  const int gpr = (N + kQGroup - 1) / kQGroup;
  const long long groups = rows * gpr;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_unpack8<T><<<seq_grid((size_t)groups, 8, 16), 256, 0, (cudaStream_t)stream>>>(groups, gpr, N, q, e, (T*)x);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  });
}

}  // extern "C"
