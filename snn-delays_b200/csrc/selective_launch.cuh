// Launches of the selective scan's kernels, shared by selective_fwd.cu and selective_bwd.cu (two
// translation units, so that they compile side by side).
#pragma once

#include "selective.cuh"

namespace delrec {

int sel_run_forward(int dtype, int L, const SelArgs& p, cudaStream_t st);
int sel_run_backward(int dtype, int L, const SelArgs& p, cudaStream_t st);

template <class T, int L, bool BWD, bool LOCAL>
static int sel_start(const SelArgs& p, cudaStream_t st) {
  const long long grid = (long long)p.tiles * p.G * p.B * p.chunks;
  if (grid > 0x7fffffffLL) return DELREC_ERR_UNSUPPORTED;
  if constexpr (BWD) {
    auto kern = k_sel_bwd<T, L, LOCAL>;
    constexpr int smem = sel_bwd_smem<T, L, LOCAL>();
    if (smem > 48 * 1024) SQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kern<<<(unsigned)grid, kSelThreads, smem, st>>>(p);
  } else {
    constexpr int smem = sel_fwd_smem<T, L, LOCAL>();
    static_assert(smem <= 48 * 1024, "needs the attribute");
    k_sel_fwd<T, L, LOCAL><<<(unsigned)grid, kSelThreads, smem, st>>>(p);
  }
  SQ_LAUNCHED();
  return DELREC_OK;
}
// the chunks' maps, their join (where time is cut), and the pass itself
template <class T, int L, bool BWD>
static int sel_pass(const SelArgs& p, cudaStream_t st) {
  if (p.chunks > 1) {
    int rc = sel_start<T, L, BWD, true>(p, st);
    if (rc) return rc;
    const size_t all = (size_t)p.B * p.N * p.S;
    k_sel_join<BWD><<<(unsigned)((all + 63) / 64), 64, 0, st>>>(p, BWD ? p.ghT : p.h0);
    SQ_LAUNCHED();
  }
  if constexpr (BWD) {   // `parts` tiles of channels a launch, each after the one before
    SelArgs q = p;
    for (q.tile0 = 0; q.tile0 < p.tiles; q.tile0 += p.parts) {
      q.tiles = std::min(p.parts, p.tiles - q.tile0);
      q.add = q.tile0 > 0;
      const int rc = sel_start<T, L, true, false>(q, st);
      if (rc) return rc;
    }
    return DELREC_OK;
  } else {
    return sel_start<T, L, false, false>(p, st);
  }
}
template <class T, bool BWD, int L = 1>
static int sel_by_l(int l, const SelArgs& p, cudaStream_t st) {
  if constexpr (4 * L <= kSelMaxS) {
    if (l != L) return sel_by_l<T, BWD, 2 * L>(l, p, st);
    return sel_pass<T, L, BWD>(p, st);
  }
  return DELREC_ERR_UNSUPPORTED;
}

}  // namespace delrec
