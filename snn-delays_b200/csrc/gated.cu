// extern "C" entry points of the gated linear recurrence: argument checks, kernel variants and
// launch shapes.  No allocation happens here.
#include <algorithm>

#include "gated_scan.cuh"
#include "seq_common.cuh"

namespace delrec {

static int check_scan(const delrec_scan* s) {
  if (!s || s->T < 1 || s->B < 1 || s->N < 1 || s->G < 1 || s->N % s->G != 0) return DELREC_ERR_ARG;
  if (s->dtype < DELREC_F32 || s->dtype > DELREC_F16) return DELREC_ERR_ARG;
  if (s->T > (1 << 30)) return DELREC_ERR_UNSUPPORTED;
  return DELREC_OK;
}

struct ScanShape {
  int V, S, P, csize;
  long long items;
  unsigned grid;
};

// May rows be read two channels at a time?  Are the inputs' rows whole 32-byte sectors, which
// may be fetched ahead without reaching past the tensor?
struct ScanAlign {
  bool two, sectors;
  int esz;
  ScanAlign(const delrec_scan* s)
      : two(s->G == s->N && s->N % 2 == 0), sectors(s->G == s->N && s->N % 64 == 0),
        esz(s->dtype == DELREC_F32 ? 4 : 2) {}
  void add(const void* ptr, long long st, long long sb) {
    if (ptr && (((uintptr_t)ptr & (2 * esz - 1)) || (st & 1) || (sb & 1))) two = false;
  }
  void input(const void* ptr, long long st, long long sb, int size) {
    add(ptr, st, sb);
    if (ptr && (((uintptr_t)ptr | (unsigned long long)(st * size) | (unsigned long long)(sb * size)) & 31))
      sectors = false;
  }
};

// V: channels per lane.  bwd: segments of 16 steps, else 16 / V.
static int scan_shape(const delrec_scan* s, ScanArgs* p, ScanShape* sh, bool bwd, int V, bool ahead) {
  p->ahead = ahead;
  p->T = s->T; p->B = s->B; p->N = s->N; p->G = s->G; p->D = s->N / s->G;
  p->decay_input = s->decay_input; p->wide = s->lengths_wide;
  for (long long st : {s->z_t, s->f_t, s->h_t, s->gh_t, s->dz_t, s->df_t})
    if (st < -0x7fffffffLL || st > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  if ((long long)s->B * s->N > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  p->split = p->D > 32;
  p->cpt = p->D == 1 || p->split ? 32 * V : 32 / p->D * p->D;
  p->tiles = (p->N + p->cpt - 1) / p->cpt;
  sh->V = V;
  sh->S = bwd ? kSeg : kSeg / V;
  const long long items = (long long)p->B * p->tiles;
  const int segs = (p->T + sh->S - 1) / sh->S;
  sh->P = segs >= 5 ? 8 : (segs >= 2 ? 4 : 1);
  // few rows: the blocks of a cluster share one row's time
  int c = 1;
  while (c < kScanCluster && items * c < 2 * kSeqSMs && sh->P * c < segs) c *= 2;
  sh->csize = c;
  if (items * c > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  sh->grid = (unsigned)(items * c);
  sh->items = items;
  return DELREC_OK;
}

static int scan_launch(void (*kern)(ScanArgs, int), ScanArgs& p, ScanShape sh, cudaStream_t st) {
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
  if (sh.csize == 1 && p.ahead) {
    // as many blocks as fit at once, each walking its items and fetching the next ahead
    int per_sm = 0;
    SQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, sh.P * 32, 0));
    cfg.gridDim.x = (unsigned)std::min<long long>(sh.grid, (long long)std::max(per_sm, 1) * kSeqSMs);
  }
  if (sh.csize > 8) {
    // 16 blocks where the GPU has room for them, else the portable 8
    int fit = 0;
    SQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (cudaOccupancyMaxActiveClusters(&fit, kern, &cfg) != cudaSuccess || fit < 1) {
      (void)cudaGetLastError();
      sh.csize = 8;
      cfg.gridDim.x = sh.grid / 2;
      at[0].val.clusterDim.x = 8;
    }
  }
  SQ_CUDA(cudaLaunchKernelEx(&cfg, kern, p, (int)sh.csize));
  SQ_LAUNCHED();
  return DELREC_OK;
}

template <class T, bool POS, int P>
static int scan_fwd_p(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
  if (p.qz)
    return scan_launch(sh.V == 2 ? k_scan_fwd<T, 2, 8, P, POS, true> : k_scan_fwd<T, 1, 16, P, POS, true>, p, sh, st);
  return scan_launch(sh.V == 2 ? k_scan_fwd<T, 2, 8, P, POS, false> : k_scan_fwd<T, 1, 16, P, POS, false>, p, sh, st);
}
template <class T, bool POS, int P>
static int scan_bwd_p(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (p.qz && sh.V == 2) return scan_launch(k_scan_bwd<T, 2, P, POS, true>, p, sh, st);
  if (p.qz) return scan_launch(k_scan_bwd<T, 1, P, POS, true>, p, sh, st);
  if constexpr (sizeof(T) == 2)
    if (sh.V == 2) return scan_launch(k_scan_bwd<T, 2, P, POS, false>, p, sh, st);
  return scan_launch(k_scan_bwd<T, 1, P, POS, false>, p, sh, st);
}
template <class T, bool POS>
static int scan_run(ScanArgs& p, const ScanShape& sh, bool bwd, cudaStream_t st) {
  switch (sh.P) {
    case 1: return bwd ? scan_bwd_p<T, POS, 1>(p, sh, st) : scan_fwd_p<T, POS, 1>(p, sh, st);
    case 4: return bwd ? scan_bwd_p<T, POS, 4>(p, sh, st) : scan_fwd_p<T, POS, 4>(p, sh, st);
    default: return bwd ? scan_bwd_p<T, POS, 8>(p, sh, st) : scan_fwd_p<T, POS, 8>(p, sh, st);
  }
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
  ScanAlign al(s);
  al.input(z, s->z_t, s->z_b, al.esz);
  al.input(f, s->f_t, s->f_b, al.esz);
  al.add(h, s->h_t, s->h_b);
  if (pack) {
    al.add(qz, 0, 0);
    al.add(qf, 0, 0);
  }
  if ((rc = scan_shape(s, &p, &sh, false, al.two ? 2 : 1, al.sectors))) return rc;
  p.z = z; p.f = f; p.h0 = h0; p.lengths = lengths; p.resets = resets; p.h = h; p.hT = hT; p.states = states;
  p.qz = qz; p.ez = ez; p.qf = qf; p.ef = ef;
  p.z_t = (int)s->z_t; p.z_b = s->z_b; p.f_t = (int)s->f_t; p.f_b = s->f_b; p.h_t = (int)s->h_t; p.h_b = s->h_b;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pos = lengths || resets;
  return by_dtype(s->dtype, [&](auto t) {
    using T = decltype(t);
    return pos ? scan_run<T, true>(p, sh, false, st) : scan_run<T, false>(p, sh, false, st);
  });
}

size_t delrec_gated_scan_backward_workspace(const delrec_scan* s) {
  if (check_scan(s)) return 0;
  const int D = s->N / s->G;
  return D > 32 ? (size_t)s->T * s->B * ((s->N + 31) / 32) * 2 * sizeof(float) : 0;
}

int delrec_gated_scan_backward(const delrec_scan* s, const void* z, const void* f, const int8_t* qz,
                               const uint8_t* ez, const int8_t* qf, const uint8_t* ef, const void* lengths,
                               const uint8_t* resets, const float* states, const void* gh, const float* ghT,
                               void* dz, void* df, float* dh0, void* ws, size_t wsb, void* stream) {
  int rc = check_scan(s);
  if (rc) return rc;
  const bool pack = qz || ez || qf || ef;
  if (!states || (pack ? !(qz && ez && qf && ef) || s->G != s->N : !z || !f)) return DELREC_ERR_ARG;
  ScanArgs p{};
  ScanShape sh;
  ScanAlign al(s);
  if (pack) {
    al.input(qz, 0, 0, 1);
    al.input(qf, 0, 0, 1);
  } else {
    al.input(z, s->z_t, s->z_b, al.esz);
    al.input(f, s->f_t, s->f_b, al.esz);
  }
  al.input(gh, s->gh_t, s->gh_b, al.esz);
  al.add(dz, s->dz_t, s->dz_b);
  al.add(df, s->df_t, s->df_b);
  if ((rc = scan_shape(s, &p, &sh, true, al.two && s->dtype != DELREC_F32 ? 2 : 1, al.sectors))) return rc;
  const size_t need = df ? delrec_gated_scan_backward_workspace(s) : 0;
  if (need && (!ws || ((uintptr_t)ws & 255) != 0 || wsb < need)) return DELREC_ERR_WORKSPACE;
  p.z = z; p.f = f; p.lengths = lengths; p.resets = resets; p.states = const_cast<float*>(states);
  p.qz = const_cast<int8_t*>(qz); p.ez = const_cast<uint8_t*>(ez);
  p.qf = const_cast<int8_t*>(qf); p.ef = const_cast<uint8_t*>(ef);
  p.gh = gh; p.ghT = ghT; p.dz = dz; p.df = df; p.dh0 = dh0; p.part = (float*)ws;
  p.z_t = (int)s->z_t; p.z_b = s->z_b; p.f_t = (int)s->f_t; p.f_b = s->f_b; p.gh_t = (int)s->gh_t; p.gh_b = s->gh_b;
  p.dz_t = (int)s->dz_t; p.dz_b = s->dz_b; p.df_t = (int)s->df_t; p.df_b = s->df_b;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pos = lengths || resets;
  return by_dtype(s->dtype, [&](auto t) {
    using T = decltype(t);
    const int r = pos ? scan_run<T, true>(p, sh, true, st) : scan_run<T, false>(p, sh, true, st);
    if (r) return r;
    if (df && p.split) {
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

}  // extern "C"
