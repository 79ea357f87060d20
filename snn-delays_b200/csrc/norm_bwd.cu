// The block norms' backward kernels.
#include "norm_launch.cuh"

namespace delrec {

int norm_run_backward(int dtype, const NormArgs& a, NormShape& s, int most, cudaStream_t st) {
  return by_dtype(dtype, [&](auto t) { return norm_run<decltype(t), true>(a, s, most, st); });
}

}  // namespace delrec
