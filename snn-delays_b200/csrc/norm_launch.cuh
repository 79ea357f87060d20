// Launches of the block-norm kernels and their choice of variant, shared by norm_fwd.cu and
// norm_bwd.cu (two translation units, so that they compile side by side).
#pragma once

#include <algorithm>

#include "block_norm.cuh"

namespace delrec {

// As many blocks as fit at once: each walks its rows, the next on its way.  Where two blocks
// or fewer fit an SM they cannot cover each other's waits, and a third row in flight pays
// (N=2048 bf16 backward 509 -> 372 us); where five fit it costs (N=512 fp32 backward 165 -> 183 us).
// most_threads: of an SM; the backward's eight streams of rows slow the memory down past 640
// threads (N=512 fp32: five blocks of 128 take 159 us, eight 182 us).
static constexpr int kNormThirdRow = 100 * 1024;   // most shared memory of a block with a third row
template <class K>
static int norm_start(K kern, int row_bytes, int most_threads, NormArgs a, NormShape& s, int most, cudaStream_t st) {
  // The limit on a launch's shared memory belongs to the kernel, not to the launch: it is always set
  // to the most that any width asks of this kernel, so that calls of other widths from other host
  // threads cannot lower it in between.
  const int full = row_bytes * kNormThreads, limit = std::max(2 * full, std::min(3 * full, kNormThirdRow));
  int per_sm = 0, smem = 0;
  for (a.slots = 2; a.slots <= 3; ++a.slots) {
    smem = a.slots * row_bytes * s.threads;
    if (smem > 40 * 1024) SQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, limit));
    SQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, s.threads, smem));
    if (per_sm > 2 || row_bytes == 0 || 3 * row_bytes * s.threads > kNormThirdRow) break;
  }
  if (a.slots > 3) a.slots = 3;
  s.grid = std::min(most, std::max(1, std::min({per_sm, 16, most_threads / s.threads})) * kSeqSMs);
  kern<<<s.grid, s.threads, smem, st>>>(a);
  SQ_LAUNCHED();
  return DELREC_OK;
}
template <class T, int V, bool BWD, int KIND, int IT = 1>
static int norm_by_it(const NormArgs& a, NormShape& s, int most, cudaStream_t st) {
  if constexpr (V * IT <= 32) {
    if (s.IT != IT) return norm_by_it<T, V, BWD, KIND, 2 * IT>(a, s, most, st);
    using Stage = NormStage<T, V, IT, BWD ? (KIND ? 5 : 4) : (KIND ? 3 : 2)>;
    if constexpr (Stage::STAGED)
      if (a.pitch > 0) {
        if constexpr (BWD) return norm_start(k_norm_bwd<T, V, IT, KIND, true>, Stage::ROW, 640, a, s, most, st);
        else return norm_start(k_norm_fwd<T, V, IT, KIND, true>, Stage::ROW, 2048, a, s, most, st);
      }
    if constexpr (BWD) return norm_start(k_norm_bwd<T, V, IT, KIND, false>, Stage::ROW, 640, a, s, most, st);
    else return norm_start(k_norm_fwd<T, V, IT, KIND, false>, Stage::ROW, 2048, a, s, most, st);
  }
  return DELREC_ERR_UNSUPPORTED;
}
template <class T, int V, bool BWD>
static int norm_by_gate(const NormArgs& a, NormShape& s, int most, cudaStream_t st) {
  if (a.kind == GATE_NONE) return norm_by_it<T, V, BWD, GATE_NONE>(a, s, most, st);
  if (a.kind == GATE_SIGMOID) return norm_by_it<T, V, BWD, GATE_SIGMOID>(a, s, most, st);
  return norm_by_it<T, V, BWD, GATE_SILU>(a, s, most, st);
}
// the widest access the tensors allow, 16 bytes at most
template <class T, bool BWD>
static int norm_run(const NormArgs& a, NormShape& s, int most, cudaStream_t st) {
  constexpr int V16 = 16 / sizeof(T), V8 = 8 / sizeof(T);
  if (s.V == V16) return norm_by_gate<T, V16, BWD>(a, s, most, st);
  if (s.V == V8) return norm_by_gate<T, V8, BWD>(a, s, most, st);
  return norm_by_gate<T, 1, BWD>(a, s, most, st);
}
}  // namespace delrec
