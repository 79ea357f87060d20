// Launches of the short convolution's kernels, shared by conv_fwd.cu and conv_bwd.cu (two
// translation units, so that they compile side by side).
#pragma once

#include <algorithm>

#include "short_conv.cuh"

namespace delrec {

int conv_run_forward(int dtype, int K, int V, const ConvArgs& a, cudaStream_t st);
int conv_run_backward(int dtype, int K, int V, const ConvArgs& a, cudaStream_t st);

template <class T, int K, int V, bool BWD>
static int conv_start(const ConvArgs& a, cudaStream_t st) {
  const long long cols = (a.N + V - 1) / V;
  if constexpr (!BWD) {
    if (a.T == 1 && !a.resets) {   // as many threads as run at once, or one to a sequence
      const int step = (int)std::min<long long>(a.B, std::max<long long>(1, kSeqSMs * 1024LL / cols));
      k_conv_step<T, K, V><<<(unsigned)((cols * step + 127) / 128), 128, 0, st>>>(a, step);
      SQ_LAUNCHED();
      return DELREC_OK;
    }
  }
  const long long blocks = (cols * a.B * a.chunks + 127) / 128;
  if (blocks > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  if constexpr (BWD) k_conv_bwd<T, K, V><<<(unsigned)blocks, 128, 0, st>>>(a);
  else k_conv_fwd<T, K, V><<<(unsigned)blocks, 128, 0, st>>>(a);
  SQ_LAUNCHED();
  return DELREC_OK;
}
template <class T, bool BWD, int K = 1>
static int conv_by_k(int k, int V, const ConvArgs& a, cudaStream_t st) {
  if constexpr (K <= kConvMaxK) {
    if (k != K) return conv_by_k<T, BWD, K + 1>(k, V, a, st);
    return V > 1 ? conv_start<T, K, 4, BWD>(a, st) : conv_start<T, K, 1, BWD>(a, st);
  }
  return DELREC_ERR_ARG;
}

}  // namespace delrec
