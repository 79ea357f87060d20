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

// What the tensors allow: sixteen-byte copies of the inputs' rows (STAGED), two channels at a time
// of the states and the codes that a forward pass writes.
struct ScanAlign {
  bool sixteen, pairs = true;
  int esz;
  ScanAlign(const delrec_scan* s) : sixteen(s->G == s->N), esz(s->dtype == DELREC_F32 ? 4 : 2) {}
  void input(const void* ptr, long long st, long long sb, int row_bytes, int size) {
    if (ptr && (((uintptr_t)ptr | (unsigned long long)(st * size) | (unsigned long long)(sb * size) |
                 (unsigned long long)row_bytes) & 15))
      sixteen = false;
  }
  // V elements at a time: pairs of a 16-bit type
  void output(const void* ptr, long long st, long long sb) {
    if (ptr && esz == 2 && (((uintptr_t)ptr & 3) || (st & 1) || (sb & 1))) sixteen = false;
  }
  void pair(const void* ptr, int size) {
    if ((uintptr_t)ptr & (2 * size - 1)) pairs = false;
  }
};

static int scan_shape(const delrec_scan* s, ScanArgs* p, ScanShape* sh, const ScanAlign& al, bool q8) {
  p->T = s->T; p->B = s->B; p->N = s->N; p->G = s->G; p->D = s->N / s->G;
  p->decay_input = s->decay_input; p->wide = s->lengths_wide;
  for (long long st : {s->z_t, s->f_t, s->h_t, s->gh_t, s->dz_t, s->df_t})
    if (st < -0x7fffffffLL || st > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  if ((long long)s->B * s->N > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  const int segs = (p->T + kSeg - 1) / kSeg;
  sh->P = segs >= 2 ? kScanWarps : 1;
  p->split = p->D >= 32;
  sh->mode = p->split ? SCAN_WIDE : (al.sixteen && p->D == 1 ? SCAN_STAGED : SCAN_DIRECT);
  // two channels to a lane (16-bit), unless that leaves SMs without a block even when a
  // cluster shares each row's time
  sh->V = sh->mode == SCAN_STAGED && s->dtype != DELREC_F32 && al.pairs &&
                  (long long)p->B * ((p->N + 63) / 64) * std::min(kScanCluster, (segs + sh->P - 1) / sh->P) >= 2 * kSeqSMs
              ? 2
              : 1;
  p->cpt = p->D == 1 || p->split ? 32 * sh->V : 32 / p->D * p->D;
  p->tiles = (p->N + p->cpt - 1) / p->cpt;
  const long long items = (long long)p->B * p->tiles;
  // a block's next item, one grid (at most all items) further, has to fit 32 bits
  if (items > 1LL << 30) return DELREC_ERR_UNSUPPORTED;
  // The blocks of a cluster share a row's time where that fills the SMs better: about two
  // blocks of 8 warps fit an SM (of the plain 16-bit backward one), the rounds they take fall
  // with the cluster's size c, and each doubling costs some 6 % in exchanges (T=1021, 408 items: c = 1 takes two rounds for
  // 1.4 blocks' work).
  const long long slots = 2 * kSeqSMs * 8 / sh->P;
  int c = 1;
  double best = 0;
  for (int k = 1, lg = 0; k <= kScanCluster && (k == 1 || sh->P * k / 2 < segs); k *= 2, ++lg) {
    const double cost = (double)((items * k + slots - 1) / slots) / k * (1 + 0.06 * lg);
    if (k == 1 || cost < best) { best = cost; c = k; }
  }
  sh->csize = c;
  // a cluster's exchange costs as much as some 16 steps: segments of 32 where there are enough,
  // and where two blocks' stages still fit an SM (16-bit)
  sh->R = c > 1 && s->dtype != DELREC_F32 && sh->mode == SCAN_STAGED && sh->V == 1 && sh->P > 1 && !q8 && segs >= 2 * sh->P * c ? 2 : 1;
  if (items * c > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  sh->grid = (unsigned)(items * c);
  return DELREC_OK;
}

}  // namespace delrec

using namespace delrec;

extern "C" {

int delrec_gated_scan_forward(const delrec_scan* s, const void* z, const void* f, const float* h0,
                              const void* lengths, const uint8_t* resets, void* h, float* hT, float* states,
                              int8_t* qz, uint8_t* ez, int8_t* qf, uint8_t* ef, uint8_t* odd, void* stream) {
  int rc = check_scan(s);
  if (rc) return rc;
  if (!z || !f || !h) return DELREC_ERR_ARG;
  const bool pack = qz || ez || qf || ef || odd;
  if (pack && (!(qz && ez && qf && ef && odd) || s->G != s->N)) return DELREC_ERR_ARG;
  ScanArgs p{};
  ScanShape sh;
  ScanAlign al(s);
  al.input(z, s->z_t, s->z_b, s->N * al.esz, al.esz);
  al.input(f, s->f_t, s->f_b, s->N * al.esz, al.esz);
  al.output(h, s->h_t, s->h_b);
  al.pair(states, sizeof(float));
  al.pair(qz, 1);
  al.pair(qf, 1);
  if ((rc = scan_shape(s, &p, &sh, al, pack))) return rc;
  p.z = z; p.f = f; p.h0 = h0; p.lengths = lengths; p.resets = resets; p.h = h; p.hT = hT; p.states = states;
  p.qz = qz; p.ez = ez; p.qf = qf; p.ef = ef; p.odd = odd;
  p.z_t = (int)s->z_t; p.z_b = s->z_b; p.f_t = (int)s->f_t; p.f_b = s->f_b; p.h_t = (int)s->h_t; p.h_b = s->h_b;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pos = lengths || resets;
  return scan_run_forward(s->dtype, p, sh, pos, st);
}

size_t delrec_gated_scan_backward_workspace(const delrec_scan* s) {
  if (check_scan(s)) return 0;
  const int D = s->N / s->G;
  return D >= 32 ? (size_t)s->T * s->B * ((s->N + 31) / 32) * 2 * sizeof(float) : 0;
}

int delrec_gated_scan_backward(const delrec_scan* s, const void* z, const void* f, const int8_t* qz,
                               const uint8_t* ez, const int8_t* qf, const uint8_t* ef, const uint8_t* odd,
                               const void* lengths,
                               const uint8_t* resets, const float* states, const void* gh, const float* ghT,
                               void* dz, void* df, float* dh0, void* ws, size_t wsb, void* stream) {
  int rc = check_scan(s);
  if (rc) return rc;
  const bool pack = qz || ez || qf || ef || odd;
  if (!states || (pack ? !(qz && ez && qf && ef && odd) || s->G != s->N : !z || !f)) return DELREC_ERR_ARG;
  ScanArgs p{};
  ScanShape sh;
  ScanAlign al(s);
  if (pack) {
    al.input(qz, 0, 0, s->N, 1);
    al.input(qf, 0, 0, s->N, 1);
  } else {
    al.input(z, s->z_t, s->z_b, s->N * al.esz, al.esz);
    al.input(f, s->f_t, s->f_b, s->N * al.esz, al.esz);
  }
  al.input(gh, s->gh_t, s->gh_b, s->N * al.esz, al.esz);
  al.output(dz, s->dz_t, s->dz_b);
  al.output(df, s->df_t, s->df_b);
  al.pair(states, sizeof(float));
  if ((rc = scan_shape(s, &p, &sh, al, pack))) return rc;
  const size_t need = df ? delrec_gated_scan_backward_workspace(s) : 0;
  if (need && (!ws || ((uintptr_t)ws & 255) != 0 || wsb < need)) return DELREC_ERR_WORKSPACE;
  p.z = z; p.f = f; p.lengths = lengths; p.resets = resets; p.states = const_cast<float*>(states);
  p.qz = const_cast<int8_t*>(qz); p.ez = const_cast<uint8_t*>(ez);
  p.qf = const_cast<int8_t*>(qf); p.ef = const_cast<uint8_t*>(ef);
  p.odd = const_cast<uint8_t*>(odd);
  p.gh = gh; p.ghT = ghT; p.dz = dz; p.df = df; p.dh0 = dh0; p.part = (float*)ws;
  p.z_t = (int)s->z_t; p.z_b = s->z_b; p.f_t = (int)s->f_t; p.f_b = s->f_b; p.gh_t = (int)s->gh_t; p.gh_b = s->gh_b;
  p.dz_t = (int)s->dz_t; p.dz_b = s->dz_b; p.df_t = (int)s->df_t; p.df_b = s->df_b;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pos = lengths || resets;
  rc = scan_run_backward(s->dtype, p, sh, pos, st);
  if (rc || !df || !p.split) return rc;
  return by_dtype(s->dtype, [&](auto t) {
    using T = decltype(t);
    {
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
