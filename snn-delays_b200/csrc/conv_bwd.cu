// The short convolution's backward kernels.
#include "conv_launch.cuh"

namespace delrec {
int conv_run_backward(int dtype, int K, int V, const ConvArgs& a, cudaStream_t st) {
  return by_dtype(dtype, [&](auto t) { return conv_by_k<decltype(t), true>(K, V, a, st); });
}
}  // namespace delrec
