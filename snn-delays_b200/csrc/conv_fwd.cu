// The short convolution's forward kernels.
#include "conv_launch.cuh"

namespace delrec {
int conv_run_forward(int dtype, int K, int V, const ConvArgs& a, cudaStream_t st) {
  return by_dtype(dtype, [&](auto t) { return conv_by_k<decltype(t), false>(K, V, a, st); });
}
}  // namespace delrec
