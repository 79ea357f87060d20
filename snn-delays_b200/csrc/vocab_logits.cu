// The logits' products of the vocabulary losses.
#include "vocab_launch.cuh"

namespace delrec {
template <int BN, int EPI>
static int run(bool f16, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st) {
  if (g.nprod > 1) return vg_start<BN, false, false, EPI, false, true, float>(A, B, g, st);
  return f16 ? vg_start<BN, false, false, EPI, true, false, float>(A, B, g, st)
             : vg_start<BN, false, false, EPI, false, false, float>(A, B, g, st);
}
int vg_logits(bool f16, int BN, bool grad, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st) {
  if (BN == 256) return grad ? run<256, VG_GRAD>(f16, A, B, g, st) : run<256, VG_STATS>(f16, A, B, g, st);
  return grad ? run<128, VG_GRAD>(f16, A, B, g, st) : run<128, VG_STATS>(f16, A, B, g, st);
}
}  // namespace delrec
