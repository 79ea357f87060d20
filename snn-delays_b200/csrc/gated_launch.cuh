// Launches of the scan kernels and their choice of variant, shared by gated_fwd.cu and
// gated_bwd.cu (two translation units, so that they compile side by side).
#pragma once

#include <algorithm>

#include "gated_scan.cuh"

namespace delrec {

static inline int scan_launch(void (*kern)(ScanArgs, int), int smem, ScanArgs& p, ScanShape sh, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(sh.grid);
  cfg.blockDim = dim3(sh.P * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  if (smem > 0) SQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = sh.csize;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = sh.csize > 1 ? 1 : 0;
  if (sh.csize == 1 && sh.mode == SCAN_STAGED) {
    // as many blocks as fit at once, each walking its items and copying the next ahead
    int per_sm = 0;
    SQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, sh.P * 32, smem));
    cfg.gridDim.x = (unsigned)std::min<long long>(sh.grid, (long long)std::max(per_sm, 1) * kSeqSMs);
  }
  if (sh.csize > 8) {
    // 16 blocks where the GPU has room for them, else the portable 8
    int fit = 0;
    SQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (cudaOccupancyMaxActiveClusters(&fit, kern, &cfg) != cudaSuccess || fit < 1) {
      (void)cudaGetLastError();
      sh.csize = 8;
      cfg.gridDim.x = sh.grid / 2;
      at[0].val.clusterDim.x = 8;
    }
  }
  SQ_CUDA(cudaLaunchKernelEx(&cfg, kern, p, (int)sh.csize));
  SQ_LAUNCHED();
  return DELREC_OK;
}

// Kernel: the direction's launcher, Kernel::run<T, V, P, R, POS, Q8, DI, MODE>(p, sh, st)
template <class Kernel, class T, bool POS, bool DI, int P, bool Q8>
static int scan_by_mode(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
  if (sh.mode == SCAN_STAGED) {
    if constexpr (sizeof(T) == 2)
      if (sh.V == 2) return Kernel::template run<T, 2, P, 1, POS, Q8, DI, SCAN_STAGED>(p, sh, st);
    if constexpr (!Q8 && P > 1 && sizeof(T) == 2)
      if (sh.R == 2) return Kernel::template run<T, 1, P, 2, POS, false, DI, SCAN_STAGED>(p, sh, st);
    return Kernel::template run<T, 1, P, 1, POS, Q8, DI, SCAN_STAGED>(p, sh, st);
  }
  if constexpr (!Q8)
    if (sh.mode == SCAN_WIDE) return Kernel::template run<T, 1, P, 1, POS, false, DI, SCAN_WIDE>(p, sh, st);
  return Kernel::template run<T, 1, P, 1, POS, Q8, DI, SCAN_DIRECT>(p, sh, st);
}
template <class Kernel, class T, bool POS, bool DI>
static int scan_by_size(ScanArgs& p, const ScanShape& sh, cudaStream_t st) {
  if (sh.P == 1)
    return p.qz ? scan_by_mode<Kernel, T, POS, DI, 1, true>(p, sh, st) : scan_by_mode<Kernel, T, POS, DI, 1, false>(p, sh, st);
  return p.qz ? scan_by_mode<Kernel, T, POS, DI, kScanWarps, true>(p, sh, st) : scan_by_mode<Kernel, T, POS, DI, kScanWarps, false>(p, sh, st);
}
template <class Kernel>
static int scan_run(int dtype, ScanArgs& p, const ScanShape& sh, bool pos, cudaStream_t st) {
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (p.decay_input)
      return pos ? scan_by_size<Kernel, T, true, true>(p, sh, st) : scan_by_size<Kernel, T, false, true>(p, sh, st);
    return pos ? scan_by_size<Kernel, T, true, false>(p, sh, st) : scan_by_size<Kernel, T, false, false>(p, sh, st);
  });
}

}  // namespace delrec
