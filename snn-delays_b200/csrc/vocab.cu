// extern "C" entry points of the vocabulary losses: argument checks, places in the workspace, the order
// of launches.  No allocation happens here.
#include <algorithm>

#include "vocab_launch.cuh"
#include "vocab_loss.cuh"

namespace delrec {

int* status_word();   // api.cu

static int check_vocab(const delrec_vocab* s) {
  if (!s || s->T < 1 || s->B < 1 || s->D < 1 || s->V < 1 || s->K < 1) return DELREC_ERR_ARG;
  if (s->dtype < DELREC_F32 || s->dtype > DELREC_F16 || s->reduction < 0 || s->reduction > 2) return DELREC_ERR_ARG;
  if (s->distill && (s->teacher_dtype < DELREC_F32 || s->teacher_dtype > DELREC_F16)) return DELREC_ERR_ARG;
  if (!s->distill && s->K != 1) return DELREC_ERR_ARG;
  if (!(s->temperature > 0.99e-6f) || !(s->temperature < 1.01e6f)) return DELREC_ERR_ARG;   // 1e-6 to 1e6
  // tiles of 256 x 128 at least, in up to 16 parts, are counted in 32 bits
  if (((long long)s->T * s->B / 256 + 1) * (s->V / 128 + 1) > (1LL << 27)) return DELREC_ERR_UNSUPPORTED;
  if (s->D > kVocabMaxD || s->K > kVocabMaxK || s->V > (1 << 30) || (long long)s->T * s->B > (1 << 24))
    return DELREC_ERR_UNSUPPORTED;
  return DELREC_OK;
}

static size_t v256(size_t v) { return (v + 255) / 256 * 256; }
struct VocabTake {
  size_t total = 0;
  size_t operator()(size_t bytes) {
    const size_t at = total;
    total += v256(bytes);
    return at;
  }
};
// what the backward pass takes over from the forward pass
struct VocabKeep {
  size_t rows, rowmap, pos, idx, p, y, lse, loss, total;
  explicit VocabKeep(const delrec_vocab* s) {
    const size_t M = (size_t)s->T * s->B, MK = M * s->K;
    VocabTake take;
    rows = take(4);
    rowmap = take(M * 4);
    pos = take(M * 4);
    idx = take(MK * 4);
    p = take(s->K > 1 ? MK * 4 : 0);
    y = take(MK * 4);
    lse = take(M * 4);
    loss = take(M * 4);
    total = take.total;
  }
};

// Positions past which the packing's blocks find the rows before their own from counts of a kernel before
// it: they read all positions before their own otherwise.
constexpr int kVocabCount = 1 << 16;
static int vocab_bn(int n) { return n <= 128 ? 128 : 256; }
// Columns of a gradient's tile: 512 where they are there (the operands of a tile cross L2 half as often
// again for twice the products), not for fp32, whose segments want two accumulators.
static int vocab_bnd(int n, int pieces) { return pieces == 1 && n > 256 && (n + 511) / 512 * 512 - n < 256 ? 512 : vocab_bn(n); }
// Parts of the reduction (kb 64-blocks) of a tm x tn grid of 256 x bn tiles: more fill the pairs of SMs
// better and cross the memory more often.  In microseconds: 0.4 a 64-block (0.65 of 512 columns), some 5 TB/s for
// the sums of the parts, written and read.
static int vocab_splits(long long tm, long long tn, int bn, long long kb, int nprod) {
  const int pairs = kSeqSMs / 2;
  int best = 1;
  double cost = 0;
  for (int k = 1; k <= 16 && (k == 1 || k * 8 <= kb); ++k) {
    const long long waves = (tm * tn * k + pairs - 1) / pairs;
    const double c = waves * ((bn == 512 ? 0.65 : 0.4) * nprod * ((kb + k - 1) / k) + 2) + (k > 1 ? (double)k * tm * 256 * tn * bn * 8 / 5e6 + 5 : 0);
    if (k == 1 || c < cost) { cost = c; best = k; }
  }
  return best;
}

struct VocabShape {
  long long M, Mp, Dp, x_piece, w_piece, g_piece;
  int pieces, gp, bnv, bnd, Vc, count; // gp pieces of G; Vc columns in each of `count` pieces of the vocabulary
  int dx_splits, dw_splits, db_runs;
  bool w_direct;                            // W is an operand as it lies
  size_t x, w, part, tab, flags, ticket, h, G, coef, inv, dx, dw, db, total;
};
// Bytes of G at once, in whole tiles of 256 columns; 512 columns of all positions where those take more (past
// 262144 positions of one 16-bit piece, 87381 of fp32): dx is read and written once a piece, so narrower ones would
// be bound by it, and take less than x's operand and dx's sums from 512 features on.
constexpr size_t kVocabBudget = 256u << 20;
static VocabShape vocab_shape(const delrec_vocab* s, bool backward) {
  VocabShape h{};
  h.M = (long long)s->T * s->B;
  h.Mp = (h.M + 255) / 256 * 256;
  h.Dp = (s->D + 7) / 8 * 8;
  h.pieces = s->dtype == DELREC_F32 ? 3 : 1;
  // G of 16-bit operands is rounded to their type: 1.4 times the error that rounding the gradients makes, where the
  // targets' entries differ.  Of few rows, where the products wait for W anyway, and where the caller wants it, a
  // second piece is kept (4096 positions distilled from 64 kept logits, 512 channels, 32768 tokens, bf16: gradients
  // 2.3e-3 -> 1.7e-3 off, the plain form's; training 503 -> 754 us; a cross entropy of 8192 positions 890 -> 1465 to 1660).
  h.gp = h.pieces == 3 ? 3 : h.M <= 512 || s->split ? 2 : 1;
  h.x_piece = h.Mp * h.Dp;
  h.w_piece = (long long)s->V * h.Dp;
  h.bnv = vocab_bn(s->V);
  h.bnd = vocab_bnd(s->D, h.pieces);
  VocabTake take;
  h.x = take((size_t)h.x_piece * h.pieces * 2);
  // whether W can be an operand as it lies is known at the call: room for its copy where it may be needed
  h.w = take(h.pieces == 1 && s->D % 8 == 0 && s->w_aligned ? 0 : (size_t)h.w_piece * h.pieces * 2);
  h.w_direct = h.pieces == 1 && s->D % 8 == 0 && s->w_aligned;
  if (!backward) {
    const long long tiles = (s->V + h.bnv - 1) / h.bnv * 2;
    h.part = take((size_t)tiles * h.Mp * sizeof(float2));
    h.tab = take(s->K > kVgFew ? (size_t)tiles * h.Mp * 4 : 0);
    h.flags = take(s->distill ? h.M : 0);
    h.ticket = take(4);
    h.h = take((size_t)h.M * 4);
  } else {
    const long long fit = std::max<long long>(512, (long long)(kVocabBudget / ((size_t)h.Mp * h.gp * 2)) / 256 * 256);
    h.count = (int)((s->V + fit - 1) / fit);
    h.Vc = (int)(((s->V + h.count - 1) / h.count + 255) / 256 * 256);
    h.count = (s->V + h.Vc - 1) / h.Vc;
    h.g_piece = h.Mp * h.Vc;
    const long long dtiles = (s->D + h.bnd - 1) / h.bnd;
    h.dx_splits = vocab_splits(h.Mp / 256, dtiles, h.bnd, std::min(h.Vc, s->V) / 64, h.gp == 3 ? 6 : h.gp);
    h.dw_splits = vocab_splits((std::min(h.Vc, s->V) + 255) / 256, dtiles, h.bnd, h.Mp / 64, h.gp == 3 ? 6 : h.gp);
    h.db_runs = (int)std::max<long long>(1, std::min<long long>(128, h.M / 32));
    h.G = take((size_t)h.g_piece * h.gp * 2);
    h.coef = take((size_t)h.M * 4);
    h.inv = take(4);
    h.dx = take((size_t)h.dx_splits * h.Mp * h.Dp * 4);
    h.dw = take(h.dw_splits > 1 ? (size_t)h.dw_splits * h.Vc * h.Dp * 4 : 0);
    h.db = take((size_t)h.db_runs * h.Vc * 4);
  }
  h.total = take.total;
  return h;
}

static VocabArgs vocab_args(const delrec_vocab* s, char* keep) {
  const VocabKeep k(s);
  VocabArgs a{};
  a.T = s->T; a.B = s->B; a.D = s->D; a.V = s->V; a.K = s->K; a.M = s->T * s->B;
  a.distill = s->distill; a.wide = s->lengths_wide; a.index_wide = s->index_wide; a.teacher = s->teacher_dtype;
  a.ignore = s->ignore_index;
  a.tau = s->temperature;
  a.scale = 1.4426950408889634f / s->temperature;
  a.x_t = s->x_t; a.x_b = s->x_b;
  a.rows = (int*)(keep + k.rows);
  a.rowmap = (int*)(keep + k.rowmap);
  a.pos = (int*)(keep + k.pos);
  a.idx = (int*)(keep + k.idx);
  a.p = s->K > 1 ? (float*)(keep + k.p) : nullptr;
  a.y = (float*)(keep + k.y);
  a.lse = (float*)(keep + k.lse);
  a.loss = (float*)(keep + k.loss);
  return a;
}

// the products of pieces, smallest first: all six of fp32's, or each piece of A with a 16-bit B
static void vg_products(VgArgs* g, int a_pieces, int b_pieces) {
  static const int pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};
  const bool six = a_pieces == 3 && b_pieces == 3;
  g->nprod = six ? 6 : a_pieces;
  for (int i = 0; i < g->nprod; ++i) {
    g->pa[i] = six ? pa[i] : a_pieces - 1 - i;
    g->pb[i] = six ? pb[i] : 0;
  }
}

// rows of x (packed) or of W as operands
static VocabPack vocab_pack_of(const delrec_vocab* s, const void* src, long long st, long long sb, int B, const int* rows,
                               const int* rowmap, long long n, long long Dp, long long piece, void* out) {
  VocabPack p{src, st, sb, n, piece, B, s->D, (int)Dp, 0, rows, rowmap, out};
  const int W = s->dtype == DELREC_F32 ? 4 : 8;
  p.vec = !((uintptr_t)src & 15) && st % W == 0 && sb % W == 0;
  return p;
}
static int vocab_pack_run(const delrec_vocab* s, const VocabPack& p, cudaStream_t st) {
  return by_dtype(s->dtype, [&](auto t) {
    k_vocab_pack<decltype(t)><<<seq_grid((size_t)(p.n + 63) / 64 * 64 * (p.Dp / 8), 256, 16), 256, 0, st>>>(p);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  });
}
static VocabPack vocab_x(const delrec_vocab* s, const VocabShape& h, const VocabArgs& a, char* ws, VgSide* X) {
  *X = VgSide{ws + h.x, s->D, h.Mp, h.Dp, h.x_piece, h.pieces};
  return vocab_pack_of(s, a.x, s->x_t, s->x_b, s->B, a.rows, a.rowmap, h.M, h.Dp, h.x_piece, ws + h.x);
}
// W as an operand: as it lies, or its copy
static int vocab_w(const delrec_vocab* s, const VocabShape& h, const VocabArgs& a, char* ws, VgSide* W, cudaStream_t st) {
  *W = VgSide{h.w_direct ? a.w : ws + h.w, s->D, s->V, h.Dp, h.w_piece, h.pieces};
  if (h.w_direct) return DELREC_OK;
  return vocab_pack_run(s, vocab_pack_of(s, a.w, s->D, 0, 1, nullptr, nullptr, s->V, h.Dp, h.w_piece, ws + h.w), st);
}

}  // namespace delrec

using namespace delrec;

extern "C" {

size_t delrec_vocab_loss_keep(const delrec_vocab* s) { return check_vocab(s) ? 0 : VocabKeep(s).total; }
size_t delrec_vocab_loss_forward_workspace(const delrec_vocab* s) { return check_vocab(s) ? 0 : vocab_shape(s, false).total; }
size_t delrec_vocab_loss_backward_workspace(const delrec_vocab* s) { return check_vocab(s) ? 0 : vocab_shape(s, true).total; }

int delrec_vocab_loss_forward(const delrec_vocab* s, const void* x, const void* w, const void* bias, const void* index,
                              const void* logits, const void* lengths, float* out, void* keep, size_t keepb, void* ws,
                              size_t wsb, void* stream) {
  const int rc0 = check_vocab(s);
  if (rc0) return rc0;
  if (!x || !w || !index || !out || (s->distill && !logits)) return DELREC_ERR_ARG;
  if (s->w_aligned && ((uintptr_t)w & 15)) return DELREC_ERR_ARG;
  const VocabShape h = vocab_shape(s, false);
  if (!keep || ((uintptr_t)keep & 255) || keepb < VocabKeep(s).total) return DELREC_ERR_WORKSPACE;
  if (!ws || ((uintptr_t)ws & 255) || wsb < h.total) return DELREC_ERR_WORKSPACE;
  char* base = (char*)ws;
  VocabArgs a = vocab_args(s, (char*)keep);
  a.x = x; a.w = w; a.bias = bias; a.index = index; a.logits = logits; a.lengths = lengths;
  a.flags = (uint8_t*)(base + h.flags);
  a.h = (float*)(base + h.h);
  a.ticket = (int*)(base + h.ticket);
  if (!(a.status = status_word())) return DELREC_ERR_CUDA;
  const cudaStream_t st = (cudaStream_t)stream;
  float* each = s->reduction == 0 ? out : nullptr;
  if (s->distill) {
    k_vocab_flags<<<(a.M + 7) / 8, 256, 0, st>>>(a);
    SQ_LAUNCHED();
  }
  int* counts = a.M > kVocabCount ? (int*)a.h : nullptr;   // (the rows' h is written later)
  if (counts) {
    k_vocab_count<<<(a.M + 1023) / 1024, 1024, 0, st>>>(a, counts);
    SQ_LAUNCHED();
  }
  k_vocab_rows<<<(a.M + 1023) / 1024, 1024, 0, st>>>(a, counts, each);
  SQ_LAUNCHED();
  VgSide X, W;
  const VocabPack pack = vocab_x(s, h, a, base, &X);
  int rc = vocab_w(s, h, a, base, &W, st);
  if (rc) return rc;
  const int halves = (s->V + h.bnv - 1) / h.bnv * 2;
  unsigned* tab = s->K > kVgFew ? (unsigned*)(base + h.tab) : nullptr;
  rc = by_dtype(s->dtype, [&](auto t) {
    using E = decltype(t);
    const int W = s->K == 1 ? 1 : s->K <= 32 ? 32 : 128, blocks = (a.M + 128 / W - 1) / (128 / W);
    int P = 128;
    while (P < s->K) P *= 2;
    const size_t smem = W == 128 ? (size_t)P * 16 : 0;
    auto kern = W == 1 ? k_vocab_targets<E, 1> : W == 32 ? k_vocab_targets<E, 32> : k_vocab_targets<E, 128>;
    kern<<<blocks + seq_grid((size_t)h.Mp * (h.Dp / 8), 128, 16), 128, smem, st>>>(a, blocks, pack, tab, h.Mp, halves, h.bnv / 2, P);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  });
  if (rc) return rc;
  VgArgs g{};
  g.rows = a.rows;
  g.M = -1; g.K = s->D; g.N = s->V; g.splits = 1; g.seg = h.pieces == 3 ? 2 : 0; g.status = a.status; g.spin_ns = 2000000000ll;
  vg_products(&g, h.pieces, h.pieces);
  g.part = (float2*)(base + h.part); g.part_ld = h.Mp;
  g.idx = a.idx; g.tab = tab; g.z = a.y; g.kept = s->K;
  g.bias = bias; g.bias_code = s->dtype; g.scale = a.scale;
  if ((rc = vg_logits(s->dtype == DELREC_F16, h.bnv, false, X, W, g, st))) return rc;
  k_vocab_lse<<<(a.M + 31) / 32, 1024, 0, st>>>(a, g.part, g.part_ld, halves, each, s->reduction == 1, each ? nullptr : out);
  SQ_LAUNCHED();
  return DELREC_OK;
}

int delrec_vocab_loss_backward(const delrec_vocab* s, const void* x, const void* w, const void* bias, const float* g_out,
                               const void* keep, size_t keepb, void* dx, void* dw, void* db, void* ws, size_t wsb,
                               void* stream) {
  const int rc0 = check_vocab(s);
  if (rc0) return rc0;
  if (!x || !w || !g_out || (db && !bias)) return DELREC_ERR_ARG;
  if (s->w_aligned && ((uintptr_t)w & 15)) return DELREC_ERR_ARG;
  const VocabShape h = vocab_shape(s, true);
  if (!keep || ((uintptr_t)keep & 255) || keepb < VocabKeep(s).total) return DELREC_ERR_WORKSPACE;
  if (!ws || ((uintptr_t)ws & 255) || wsb < h.total) return DELREC_ERR_WORKSPACE;
  char* base = (char*)ws;
  VocabArgs a = vocab_args(s, (char*)const_cast<void*>(keep));
  a.x = x; a.w = w; a.bias = bias;
  if (!(a.status = status_word())) return DELREC_ERR_CUDA;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool f16 = s->dtype == DELREC_F16;
  float *coef = (float*)(base + h.coef), *inv = (float*)(base + h.inv);
  k_vocab_coef<<<1, 1024, 0, st>>>(a, s->reduction, g_out, coef, inv);
  SQ_LAUNCHED();
  VgSide X, W;
  int rc = vocab_pack_run(s, vocab_x(s, h, a, base, &X), st);
  if (rc || (rc = vocab_w(s, h, a, base, &W, st))) return rc;
  const VgSide G{base + h.G, h.Vc, h.Mp, h.Vc, h.g_piece, h.gp};
  const long long MK = (long long)a.M * a.K;
  for (int c = 0; c < h.count; ++c) {
    const int v0 = c * h.Vc, n = std::min(h.Vc, s->V - v0);
    VgArgs g{};
    g.rows = a.rows; g.status = a.status; g.spin_ns = 2000000000ll;
    vg_products(&g, h.gp, h.pieces);
    {   // G = c softmax(z), then c (softmax(z) - p) at the targets
      VgArgs q = g;
      vg_products(&q, h.pieces, h.pieces);
      q.M = -1; q.K = s->D; q.N = n; q.splits = 1; q.seg = h.pieces == 3 ? 2 : 0; q.b_mn = v0;
      q.bias = bias; q.bias_code = s->dtype; q.scale = a.scale;
      q.lse = a.lse; q.coef = coef; q.G = base + h.G; q.g_ld = h.Vc; q.g_piece = h.g_piece; q.pieces = h.gp;
      if ((rc = vg_logits(f16, h.bnv, true, X, W, q, st))) return rc;
      const unsigned blocks = (unsigned)((MK + 255) / 256);
      if (f16) k_vocab_patch<__half><<<blocks, 256, 0, st>>>(a, coef, v0, n, (__half*)(base + h.G), h.Vc, h.g_piece, h.gp);
      else k_vocab_patch<__nv_bfloat16><<<blocks, 256, 0, st>>>(a, coef, v0, n, (__nv_bfloat16*)(base + h.G), h.Vc, h.g_piece, h.gp);
      SQ_LAUNCHED();
    }
    const int seg = h.pieces == 3 ? 8 : 0;
    if (dw) {   // rows v0.. of G^T x
      VgArgs q = g;
      q.M = n; q.K = -1; q.N = s->D; q.splits = h.dw_splits; q.seg = seg; q.inv = inv;
      if (h.dw_splits > 1) {
        q.plane = (float*)(base + h.dw); q.plane_ld = h.Dp; q.plane_split = (long long)h.Vc * h.Dp;
      } else {
        q.out = dw; q.out_ld = s->D; q.out0 = v0;
      }
      if ((rc = vg_weights(s->dtype, h.bnd, G, X, q, st))) return rc;
      if (h.dw_splits > 1) {
        rc = by_dtype(s->dtype, [&](auto t) {
          using E = decltype(t);
          k_vocab_planes<E><<<seq_grid((size_t)n * ((s->D + 3) / 4), 256, 8), 256, 0, st>>>(
              n, s->D, nullptr, q.plane, q.plane_ld, q.plane_split, q.splits, inv, (E*)dw + (long long)v0 * s->D);
          SQ_LAUNCHED();
          return (int)DELREC_OK;
        });
        if (rc) return rc;
      }
    }
    if (dx) {   // += G W[v0..]
      VgArgs q = g;
      q.M = -1; q.K = n; q.N = s->D; q.splits = h.dx_splits; q.seg = seg; q.b_k = v0;
      q.plane = (float*)(base + h.dx); q.plane_ld = h.Dp; q.plane_split = h.Mp * h.Dp; q.accumulate = c > 0;
      if ((rc = vg_inputs(f16, h.bnd, G, W, q, st))) return rc;
    }
    if (db) {
      float* part = (float*)(base + h.db);
      const dim3 grid((n + 1023) / 1024, h.db_runs);
      const auto sum = [&](auto e, auto pieces) {
        using E = decltype(e);
        k_vocab_db_part<E, decltype(pieces)::value><<<grid, 128, 0, st>>>(a.rows, (const E*)(base + h.G), n, h.Vc, h.g_piece, part);
      };
      using One = std::integral_constant<int, 1>;
      using Two = std::integral_constant<int, 2>;
      using Three = std::integral_constant<int, 3>;
      if (f16) h.gp == 1 ? sum(__half(), One()) : sum(__half(), Two());
      else h.gp == 1 ? sum(__nv_bfloat16(), One()) : h.gp == 2 ? sum(__nv_bfloat16(), Two()) : sum(__nv_bfloat16(), Three());
      SQ_LAUNCHED();
      rc = by_dtype(s->dtype, [&](auto t) {
        using E = decltype(t);
        k_vocab_db<E><<<(n + 255) / 256, 256, 0, st>>>(part, n, h.db_runs, inv, (E*)db + v0);
        SQ_LAUNCHED();
        return (int)DELREC_OK;
      });
      if (rc) return rc;
    }
  }
  if (!dx) return DELREC_OK;
  return by_dtype(s->dtype, [&](auto t) {
    using E = decltype(t);
    k_vocab_planes<E><<<seq_grid((size_t)h.M * ((s->D + 3) / 4), 256, 8), 256, 0, st>>>(
        h.M, s->D, a.pos, (const float*)(base + h.dx), h.Dp, h.Mp * h.Dp, h.dx_splits, inv, (E*)dx);
    SQ_LAUNCHED();
    return (int)DELREC_OK;
  });
}

}  // extern "C"
