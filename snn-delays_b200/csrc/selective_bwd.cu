// The selective scan's backward kernels.
#include "selective_launch.cuh"

namespace delrec {
int sel_run_backward(int dtype, int L, const SelArgs& p, cudaStream_t st) {
  return by_dtype(dtype, [&](auto t) { return sel_by_l<decltype(t), true>(L, p, st); });
}
}  // namespace delrec
