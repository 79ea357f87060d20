// The block norms' forward kernels.
#include "norm_launch.cuh"

namespace delrec {

int norm_run_forward(int dtype, const NormArgs& a, NormShape& s, int most, cudaStream_t st) {
  return by_dtype(dtype, [&](auto t) { return norm_run<decltype(t), false>(a, s, most, st); });
}

}  // namespace delrec
