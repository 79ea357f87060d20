// extern "C" entry points of the selective scan: argument checks, launch shapes, the step.  No
// allocation happens here.
#include <algorithm>

#include "selective_launch.cuh"

namespace delrec {

static int check_selective(const delrec_selective* s) {
  if (!s || s->T < 1 || s->B < 1 || s->N < 1 || s->S < 1 || s->G < 1 || s->N % s->G != 0) return DELREC_ERR_ARG;
  if (s->dtype < DELREC_F32 || s->dtype > DELREC_F16) return DELREC_ERR_ARG;
  if (s->S > kSelMaxS || s->T > (1 << 30)) return DELREC_ERR_UNSUPPORTED;
  // rows (B N) and their states are counted in 32 bits
  if ((long long)s->B * s->N > 0x7fffffffLL || (long long)s->N * s->S > 0x7fffffffLL ||
      (long long)s->B * s->N * s->S > (1LL << 38))
    return DELREC_ERR_UNSUPPORTED;
  return DELREC_OK;
}

static int sel_lanes(int S) {
  int L = 1;
  while (4 * L < S) L *= 2;
  return L;
}
// Lanes to a channel in the scan: a block's 256 / L channels are no more than a narrow group needs
// (each lane then lays out fewer), up to the 8 lanes whose kernels fit the SM best.
static int sel_scan_lanes(int S, int Dg) {
  int L = sel_lanes(S);
  while (L < 8 && 128 / L >= Dg) L *= 2;
  return L;
}

struct SelShape {
  int L, tiles, chunks, steps;
  int parts;                      // tiles of a backward launch
};
// Time is cut into chunks of at least 64 steps where that fills the SMs better: `slots` blocks run at
// once, so c chunks take ceil(blocks c / slots) / c of a sequence's time, and the maps that go before
// them `more` as much again (T=1021 B=24 N=520 S=24: 480 blocks for 444 slots, two rounds uncut).  Past
// four rounds uncut there is nothing to gain.
static SelShape sel_shape(const delrec_selective* s, int slots, double more) {
  SelShape h{};
  const int Dg = s->N / s->G;
  h.L = sel_scan_lanes(s->S, Dg);
  const int CH = 256 / h.L;
  h.tiles = (Dg + CH - 1) / CH;
  const long long base = (long long)h.tiles * s->G * s->B;
  // of a padded batch's k chunks some (k + 1) / 2 hold steps, and the other blocks leave at once
  const auto rounds = [&](long long k) {
    const long long blocks = s->ragged ? base * (k + 1) / 2 : base * k;
    return (double)((blocks + slots - 1) / slots);
  };
  int chunks = 1;
  double best = rounds(1);
  if (base < 4LL * slots)
    for (int k = 2; k <= s->T / 64 && k <= 1024; ++k) {
      const double cost = rounds(k) / k * (1 + more) * (1 + 0.001 * k);
      if (cost < best) { best = cost; chunks = k; }
    }
  h.steps = ((s->T + chunks - 1) / chunks + kSelSeg - 1) / kSelSeg * kSelSeg;
  h.chunks = (s->T + h.steps - 1) / h.steps;
  // Sums of dB and dC wait in one place a tile of channels: (tiles, T, B, G, S) floats twice.  Where those are more
  // than the states kept for the pass (S > 64: 8 channels to a tile; SelThread::PARTS), a launch takes a part of the tiles and the next
  // one adds to its sums, if each still fills the GPU eight times (N = 2048, S = 128, T = 64, B = 256: 4.4 -> 2.2 GB,
  // 10.3 -> 10.5 ms; as few places as fill the GPU, 14 of 256: 0.6 GB, 11.0 ms).
  const long long full = (8LL * slots + (long long)s->G * s->B - 1) / ((long long)s->G * s->B);
  h.parts = (int)std::min<long long>(h.tiles, std::max<long long>(full, (Dg + 15) / 16));
  const int launches = (h.tiles + h.parts - 1) / h.parts;
  h.parts = (h.tiles + launches - 1) / launches;
  return h;
}
static SelShape sel_fwd_shape(const delrec_selective* s) { return sel_shape(s, kSeqSMs * 5, 0.6); }
static SelShape sel_bwd_shape(const delrec_selective* s) { return sel_shape(s, kSeqSMs * 3, 0.35); }

static size_t al256(size_t v) { return (v + 255) / 256 * 256; }
struct SelPlan {   // places in the workspace
  size_t loc = 0, sumd = 0, cut = 0, dA = 0, dD = 0, db = 0, dB = 0, dC = 0, total = 0;
  size_t take(size_t bytes) {
    const size_t at = total;
    total += al256(bytes);
    return at;
  }
  void chunks(const delrec_selective* s, const SelShape& h) {
    if (h.chunks < 2) return;
    const size_t rows = (size_t)h.chunks * s->B;
    loc = take(rows * s->N * s->S * 4);
    sumd = take(rows * s->N * 4);
    cut = take(rows);
  }
};
static SelPlan sel_fwd_plan(const delrec_selective* s) {
  SelPlan w;
  w.chunks(s, sel_fwd_shape(s));
  return w;
}
static SelPlan sel_bwd_plan(const delrec_selective* s) {
  const SelShape h = sel_bwd_shape(s);
  SelPlan w;
  w.chunks(s, h);
  const size_t rows = (size_t)h.chunks * s->B, bc = s->no_bc ? 0 : (size_t)h.parts * s->T * s->B * s->G * s->S;
  w.dA = w.take(rows * s->N * s->S * 4);
  w.dD = w.take(rows * s->N * 4);
  w.db = w.take(rows * s->N * 4);
  w.dB = w.take(bc * 4);
  w.dC = w.take(bc * 4);
  return w;
}

// May all these tensors be read four, two elements at a time?
struct SelAlign {
  int esz, vec;
  SelAlign(const delrec_selective* s) : esz(s->dtype == DELREC_F32 ? 4 : 2), vec(s->N / s->G % 4 == 0 ? 4 : s->N / s->G % 2 == 0 ? 2 : 1) {}
  bool fits(int V, const void* p, long long st, long long sb) const {
    return !p || !(((uintptr_t)p % (V * esz)) || st % V || sb % V);
  }
  void add(const void* p, long long st, long long sb) {
    while (vec > 1 && !fits(vec, p, st, sb)) vec /= 2;
  }
  bool states(const delrec_selective* s, const void* Bm, const void* Cm) const {
    return s->S % 4 == 0 && fits(4, Bm, s->bm_t, s->bm_b) && fits(4, Cm, s->cm_t, s->cm_b);
  }
};

static SelArgs sel_args(const delrec_selective* s, const SelShape& h, const SelPlan& w, char* ws) {
  SelArgs p{};
  p.T = s->T; p.B = s->B; p.N = s->N; p.S = s->S; p.G = s->G; p.Dg = s->N / s->G;
  p.softplus = s->softplus; p.wide = s->lengths_wide;
  p.chunks = h.chunks; p.steps = h.steps; p.tiles = h.tiles; p.parts = h.parts;
  p.x_t = s->x_t; p.x_b = s->x_b; p.dt_t = s->dt_t; p.dt_b = s->dt_b; p.u_t = s->u_t; p.u_b = s->u_b;
  p.y_t = s->y_t; p.y_b = s->y_b; p.bm_t = s->bm_t; p.bm_b = s->bm_b; p.cm_t = s->cm_t; p.cm_b = s->cm_b;
  p.gy_t = s->gy_t; p.gy_b = s->gy_b; p.dx_t = s->dx_t; p.dx_b = s->dx_b; p.ddt_t = s->ddt_t; p.ddt_b = s->ddt_b;
  p.du_t = s->du_t; p.du_b = s->du_b;
  if (h.chunks > 1) {
    p.loc = (float*)(ws + w.loc); p.sumd = (float*)(ws + w.sumd); p.cut = (uint8_t*)(ws + w.cut);
  }
  return p;
}

}  // namespace delrec

using namespace delrec;

extern "C" {

size_t delrec_selective_forward_workspace(const delrec_selective* s) {
  return check_selective(s) ? 0 : sel_fwd_plan(s).total;
}

int delrec_selective_forward(const delrec_selective* s, const void* x, const void* dt, const float* A, const void* Bm,
                             const void* Cm, const float* D, const void* gate, const float* dt_bias, const float* h0,
                             const void* lengths, const uint8_t* resets, void* y, float* hT, float* states, void* ws,
                             size_t wsb, void* stream) {
  const int rc = check_selective(s);
  if (rc) return rc;
  if (!x || !dt || !A || !Bm || !Cm || !y || !hT) return DELREC_ERR_ARG;
  if (s->S % 4 == 0 && (((uintptr_t)hT | (uintptr_t)states) & 15)) return DELREC_ERR_ARG;
  const SelShape h = sel_fwd_shape(s);
  const SelPlan w = sel_fwd_plan(s);
  if (w.total && (!ws || ((uintptr_t)ws & 255) != 0 || wsb < w.total)) return DELREC_ERR_WORKSPACE;
  SelArgs p = sel_args(s, h, w, (char*)ws);
  p.x = x; p.dt = dt; p.A = A; p.Bm = Bm; p.Cm = Cm; p.D = D; p.gate = gate; p.bias = dt_bias; p.h0 = h0;
  p.lengths = lengths; p.resets = resets; p.y = y; p.hT = hT; p.states = states;
  SelAlign al(s);
  al.add(x, s->x_t, s->x_b);
  al.add(dt, s->dt_t, s->dt_b);
  al.add(gate, s->u_t, s->u_b);
  al.add(y, s->y_t, s->y_b);
  p.vec = al.vec;
  p.bcvec = al.states(s, Bm, Cm);
  return sel_run_forward(s->dtype, h.L, p, (cudaStream_t)stream);
}

size_t delrec_selective_backward_workspace(const delrec_selective* s) {
  return check_selective(s) ? 0 : sel_bwd_plan(s).total;
}

int delrec_selective_backward(const delrec_selective* s, const void* x, const void* dt, const float* A, const void* Bm,
                              const void* Cm, const float* D, const void* gate, const float* dt_bias,
                              const void* lengths, const uint8_t* resets, const float* states, const void* gy,
                              const float* ghT, void* dx, void* ddt, float* dA, void* dB, void* dC, float* dD,
                              void* dgate, float* ddt_bias, float* dh0, void* ws, size_t wsb, void* stream) {
  const int rc = check_selective(s);
  if (rc) return rc;
  if (!x || !dt || !A || !Bm || !Cm || !states || (dgate && !gate) || (s->no_bc && (dB || dC))) return DELREC_ERR_ARG;
  if (s->S % 4 == 0 && (((uintptr_t)dh0) & 15)) return DELREC_ERR_ARG;
  const SelShape h = sel_bwd_shape(s);
  const SelPlan w = sel_bwd_plan(s);
  if (!ws || ((uintptr_t)ws & 255) != 0 || wsb < w.total) return DELREC_ERR_WORKSPACE;
  char* base = (char*)ws;
  SelArgs p = sel_args(s, h, w, base);
  p.x = x; p.dt = dt; p.A = A; p.Bm = Bm; p.Cm = Cm; p.D = D; p.gate = gate; p.bias = dt_bias;
  p.lengths = lengths; p.resets = resets; p.states = const_cast<float*>(states); p.gy = gy; p.ghT = ghT;
  p.dx = dx; p.ddt = ddt; p.dgate = dgate; p.dh0 = dh0;
  p.dA = dA ? (float*)(base + w.dA) : nullptr;
  p.dD = dD ? (float*)(base + w.dD) : nullptr;
  p.db = ddt_bias ? (float*)(base + w.db) : nullptr;
  p.dB = dB ? (float*)(base + w.dB) : nullptr;
  p.dC = dC ? (float*)(base + w.dC) : nullptr;
  if (!dB && !dC) p.parts = p.tiles;
  SelAlign al(s);
  al.add(x, s->x_t, s->x_b);
  al.add(dt, s->dt_t, s->dt_b);
  al.add(gate, s->u_t, s->u_b);
  al.add(gy, s->gy_t, s->gy_b);
  al.add(dx, s->dx_t, s->dx_b);
  al.add(ddt, s->ddt_t, s->ddt_b);
  al.add(dgate, s->du_t, s->du_b);
  p.vec = al.vec;
  p.bcvec = al.states(s, Bm, Cm);
  const cudaStream_t st = (cudaStream_t)stream;
  int r = sel_run_backward(s->dtype, h.L, p, st);
  if (r) return r;
  const long long parts = (long long)h.chunks * s->B;
  const auto sum = [&](long long cols, const float* part, float* out) {
    if (!out) return (int)DELREC_OK;
    k_sel_sum<<<(unsigned)((cols + 31) / 32), 1024, 0, st>>>(cols, parts, part, out);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  };
  if ((r = sum((long long)s->N * s->S, p.dA, dA)) || (r = sum(s->N, p.dD, dD)) || (r = sum(s->N, p.db, ddt_bias)))
    return r;
  if (dB || dC) {
    const long long cols = (long long)s->T * s->B * s->G * s->S, blocks = (cols + 255) / 256;
    if (blocks > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
    return by_dtype(s->dtype, [&](auto t) {
      using E = decltype(t);
      k_sel_bc<E><<<(unsigned)blocks, 256, 0, st>>>(cols, h.parts, p.dB, p.dC, (E*)dB, (E*)dC);
      SQ_LAUNCHED();
      return (int)DELREC_OK;
    });
  }
  return DELREC_OK;
}

int delrec_selective_step(const delrec_selective* s, const void* x, const void* dt, const float* A, const void* Bm,
                          const void* Cm, const float* D, const void* gate, const float* dt_bias, const float* state,
                          const uint8_t* active, void* y, float* next, void* stream) {
  const int rc = check_selective(s);
  if (rc) return rc;
  if (s->T != 1 || !x || !dt || !A || !Bm || !Cm || !y || !next) return DELREC_ERR_ARG;
  SelStep p{};
  p.B = s->B; p.N = s->N; p.S = s->S; p.G = s->G; p.softplus = s->softplus;
  p.four = s->S % 4 == 0 && !(((uintptr_t)state | (uintptr_t)next) & 15);
  p.x = x; p.dt = dt; p.Bm = Bm; p.Cm = Cm; p.gate = gate; p.A = A; p.D = D; p.bias = dt_bias; p.state = state;
  p.active = active; p.y = y; p.next = next;
  p.x_b = s->x_b; p.dt_b = s->dt_b; p.u_b = s->u_b; p.bm_b = s->bm_b; p.cm_b = s->cm_b;
  const cudaStream_t st = (cudaStream_t)stream;
  p.Dg = s->N / s->G;
  const SelAlign al(s);
  p.bcvec = al.states(s, Bm, Cm);
  const int L = sel_lanes(s->S), L8 = L >= 4 ? L / 2 : L;
  const long long threads = kSeqSMs * 1024LL, NL = (long long)s->N * L8;
  if (state && p.four && s->B * NL > threads) {   // more than run at once: eight states to a lane from S = 9 on
    const int rows = (int)std::max<long long>(1, threads / NL);
    const long long blocks = (rows * NL + 255) / 256;
    if (blocks > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
    return by_dtype(s->dtype, [&](auto t) {
      using E = decltype(t);
      void (*kern)(SelStep, int) = L == 1 ? k_sel_steps<E, 1, 4> : L == 2 ? k_sel_steps<E, 2, 4> : L == 4 ? k_sel_steps<E, 2, 8>
                                 : L == 8 ? k_sel_steps<E, 4, 8> : L == 16 ? k_sel_steps<E, 8, 8> : k_sel_steps<E, 16, 8>;
      kern<<<(unsigned)blocks, 256, 0, st>>>(p, rows);
      SQ_LAUNCHED();
      return (int)DELREC_OK;
    });
  }
  const long long blocks = ((long long)s->B * s->N * L + 255) / 256;
  if (blocks > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  return by_dtype(s->dtype, [&](auto t) {
    using E = decltype(t);
    void (*kern)(SelStep) = L == 1 ? k_sel_step<E, 1> : L == 2 ? k_sel_step<E, 2> : L == 4 ? k_sel_step<E, 4>
                          : L == 8 ? k_sel_step<E, 8> : L == 16 ? k_sel_step<E, 16> : k_sel_step<E, 32>;
    kern<<<(unsigned)blocks, 256, 0, st>>>(p);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  });
}

}  // extern "C"
