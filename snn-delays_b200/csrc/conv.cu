// extern "C" entry points of the short causal convolution: argument checks, kernel variants and
// launch shapes.  No allocation happens here.
#include <algorithm>

#include "conv_launch.cuh"

namespace delrec {

static int check_conv(const delrec_conv* s) {
  if (!s || s->T < 1 || s->B < 1 || s->N < 1 || s->K < 1 || s->K > kConvMaxK) return DELREC_ERR_ARG;
  if (s->dtype < DELREC_F32 || s->dtype > DELREC_F16 || s->act < CONV_NONE || s->act > CONV_SILU) return DELREC_ERR_ARG;
  if (s->lengths_kind < 0 || s->lengths_kind > 2) return DELREC_ERR_ARG;
  if (s->T > (1 << 30)) return DELREC_ERR_UNSUPPORTED;
  return DELREC_OK;
}

// May all these tensors be read V elements at a time?
struct ConvAlign {
  int esz, V;
  bool ok;
  ConvAlign(int esz_, int V_, int N) : esz(esz_), V(V_), ok(N % V_ == 0) {}
  void add(const void* p, long long st, long long sb) {
    if (p && (((uintptr_t)p % (V * esz)) || st % V || sb % V)) ok = false;
  }
};

// Four channels to a thread: eight 16-bit ones take twice the registers, and a quarter of the warps
// then fit an SM (T=250 B=256 N=512 K=4 bf16 forward 62 us, four 41).  One to a thread where N is no multiple of
// four or a tensor lies odd: the same with N=510, 56 us forward and 121 backward instead of 42 and 90 (fp32 73 and 137
// instead of 53 and 135).
static constexpr int kConvWidth = 4;
// Chunks of time: threads of four channels for `per_sm` an SM, as many as fit at once, whose rows in
// flight cover the memory's latency; at least 8 (K - 1) rows each, of which the rows in front of (and
// behind) it are read twice.
static void conv_shape(const delrec_conv* s, int per_sm, ConvArgs* a) {
  const long long per = (long long)((s->N + kConvWidth - 1) / kConvWidth) * s->B;
  const long long want = kSeqSMs * (long long)per_sm / per;
  const int least = std::max(8 * (s->K - 1), 16);
  const int most = std::max(1, s->T / least);
  a->chunks = (int)std::max<long long>(1, std::min<long long>(want, most));
  a->steps = (s->T + a->chunks - 1) / a->chunks;
  a->chunks = (s->T + a->steps - 1) / a->steps;
}
static constexpr int kConvFwd = 768, kConvBwd = 512;   // threads an SM
static size_t conv_ws(const delrec_conv* s) {
  ConvArgs a{};
  conv_shape(s, kConvBwd, &a);
  return (size_t)a.chunks * s->B * (s->K + 1) * s->N * sizeof(float);
}

}  // namespace delrec

using namespace delrec;

extern "C" {

int delrec_short_conv_forward(const delrec_conv* s, const void* x, const float* w, const float* bias,
                              const void* state, const void* lengths, const uint8_t* resets, void* y, void* next,
                              void* stream) {
  const int rc = check_conv(s);
  if (rc) return rc;
  if (!x || !w || !y) return DELREC_ERR_ARG;
  ConvArgs a{};
  a.T = s->T; a.B = s->B; a.N = s->N; a.act = s->act; a.kind = s->lengths_kind;
  a.x = x; a.w = w; a.bias = bias; a.state = state; a.lengths = lengths; a.resets = resets; a.y = y; a.next = next;
  a.x_t = s->x_t; a.x_b = s->x_b; a.y_t = s->y_t; a.y_b = s->y_b;
  const int esz = s->dtype == DELREC_F32 ? 4 : 2;
  ConvAlign al(esz, kConvWidth, s->N);
  al.add(x, s->x_t, s->x_b);
  al.add(y, s->y_t, s->y_b);
  al.add(state, 0, 0);
  al.add(next, 0, 0);
  if (s->T == 1 && (uintptr_t)w % 16) al.ok = false;   // k_conv_step takes the filters in fours
  conv_shape(s, kConvFwd, &a);
  return conv_run_forward(s->dtype, s->K, al.ok ? al.V : 1, a, (cudaStream_t)stream);
}

size_t delrec_short_conv_backward_workspace(const delrec_conv* s) { return check_conv(s) ? 0 : conv_ws(s); }

int delrec_short_conv_backward(const delrec_conv* s, const void* x, const float* w, const float* bias,
                               const void* state, const void* lengths, const uint8_t* resets, const void* gy,
                               const void* gs, void* dx, void* ds, float* dw, float* db, void* ws, size_t wsb,
                               void* stream) {
  const int rc = check_conv(s);
  if (rc) return rc;
  if (!x || !w) return DELREC_ERR_ARG;
  const bool sums = dw || db;
  if (sums && (!ws || ((uintptr_t)ws & 255) != 0 || wsb < conv_ws(s))) return DELREC_ERR_WORKSPACE;
  ConvArgs a{};
  a.T = s->T; a.B = s->B; a.N = s->N; a.act = s->act; a.kind = s->lengths_kind;
  a.x = x; a.w = w; a.bias = bias; a.state = state; a.lengths = lengths; a.resets = resets;
  a.gy = gy; a.gs = gs; a.dx = dx; a.ds = ds; a.part = sums ? (float*)ws : nullptr;
  a.x_t = s->x_t; a.x_b = s->x_b; a.gy_t = s->gy_t; a.gy_b = s->gy_b; a.dx_t = s->dx_t; a.dx_b = s->dx_b;
  ConvAlign al(s->dtype == DELREC_F32 ? 4 : 2, kConvWidth, s->N);
  al.add(x, s->x_t, s->x_b);
  al.add(gy, s->gy_t, s->gy_b);
  al.add(dx, s->dx_t, s->dx_b);
  al.add(state, 0, 0);
  al.add(gs, 0, 0);
  al.add(ds, 0, 0);
  const cudaStream_t st = (cudaStream_t)stream;
  conv_shape(s, kConvBwd, &a);
  const int r = conv_run_backward(s->dtype, s->K, al.ok ? al.V : 1, a, st);
  if (r || !sums) return r;
  k_conv_dw<<<dim3((s->N + 31) / 32, s->K + 1), 1024, 0, st>>>(s->N, s->K, a.chunks * s->B, (const float*)ws, dw, db);
  SQ_LAUNCHED();
  return DELREC_OK;
}

}  // extern "C"
