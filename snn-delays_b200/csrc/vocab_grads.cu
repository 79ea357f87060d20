// The products of the vocabulary losses' gradients.
#include "vocab_launch.cuh"

namespace delrec {
template <int BN>
static int weights(int dtype, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st) {
  if (dtype == DELREC_F16) return vg_start<BN, true, true, VG_OUT, true, false, __half>(A, B, g, st);
  if (dtype == DELREC_BF16) return vg_start<BN, true, true, VG_OUT, false, false, __nv_bfloat16>(A, B, g, st);
  if constexpr (BN < 512) return vg_start<BN, true, true, VG_OUT, false, false, float>(A, B, g, st);
  return DELREC_ERR_ARG;   // fp32's segments want two accumulators
}
int vg_weights(int dtype, int BN, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st) {
  return BN == 512 ? weights<512>(dtype, A, B, g, st) : BN == 256 ? weights<256>(dtype, A, B, g, st) : weights<128>(dtype, A, B, g, st);
}
template <int BN>
static int inputs(bool f16, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st) {
  return f16 ? vg_start<BN, false, true, VG_OUT, true, false, float>(A, B, g, st)
             : vg_start<BN, false, true, VG_OUT, false, false, float>(A, B, g, st);
}
int vg_inputs(bool f16, int BN, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st) {
  return BN == 512 ? inputs<512>(f16, A, B, g, st) : BN == 256 ? inputs<256>(f16, A, B, g, st) : inputs<128>(f16, A, B, g, st);
}
}  // namespace delrec
