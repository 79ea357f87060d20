// The selective scan's forward kernels.
#include "selective_launch.cuh"

namespace delrec {
int sel_run_forward(int dtype, int L, const SelArgs& p, cudaStream_t st) {
  return by_dtype(dtype, [&](auto t) { return sel_by_l<decltype(t), false>(L, p, st); });
}
}  // namespace delrec
