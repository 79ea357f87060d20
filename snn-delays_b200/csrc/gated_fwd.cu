// The gated scan's forward kernels.
#include "gated_launch.cuh"

namespace delrec {

struct ScanForward {
  template <class T, int V, int P, int R, bool POS, bool PACK, bool DI, int MODE>
  static int run(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
    return scan_launch(k_scan_fwd<T, V, P, R, POS, PACK, DI, MODE>, ScanFwd<T, V, P, R, POS, PACK, MODE>::SMEM, p, sh, st);
  }
};
int scan_run_forward(int dtype, ScanArgs& p, const ScanShape& sh, bool pos, cudaStream_t st) {
  return scan_run<ScanForward>(dtype, p, sh, pos, st);
}

}  // namespace delrec
