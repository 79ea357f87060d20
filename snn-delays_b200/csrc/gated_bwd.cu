// The gated scan's backward kernels.
#include "gated_launch.cuh"

namespace delrec {

struct ScanBackward {
  template <class T, int V, int P, int R, bool POS, bool B8, bool DI, int MODE>
  static int run(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
    return scan_launch(k_scan_bwd<T, V, P, R, POS, B8, DI, MODE>, ScanBwd<T, V, P, R, B8, MODE>::SMEM, p, sh, st);
  }
};
int scan_run_backward(int dtype, ScanArgs& p, const ScanShape& sh, bool pos, cudaStream_t st) {
  return scan_run<ScanBackward>(dtype, p, sh, pos, st);
}

}  // namespace delrec
