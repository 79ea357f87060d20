// Launches of the vocabulary losses' matrix products, shared by vocab.cu and the translation units of
// the kernels' variants (so that they compile side by side).
#pragma once

#include "vocab_gemm.cuh"

namespace delrec {

// one operand: pieces of `rows` x `cols` 16-bit values of pitch ld, `piece` elements apart
struct VgSide {
  const void* p;
  long long cols, rows, ld, piece;
  int pieces;
};
int vg_logits(bool f16, int BN, bool grad, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st);
// dtype: of the result where it is written in the element type
int vg_weights(int dtype, int BN, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st);
int vg_inputs(bool f16, int BN, const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st);

static bool vg_map(CUtensorMap* m, const VgSide& s, bool f16, int box_rows) {
  TmapEncodeFn fn = tmap_encoder();
  if (!fn || !s.p || s.cols < 1 || s.rows < 1 || ((uintptr_t)s.p & 15) || (s.ld * 2 & 15) || (s.piece * 2 & 15)) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)s.cols, (cuuint64_t)s.rows, (cuuint64_t)s.pieces};
  const cuuint64_t strides[2] = {(cuuint64_t)(s.ld * 2), (cuuint64_t)(s.piece * 2)};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
  return fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(s.p), dims,
            strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool AMN, bool BMN, int EPI, bool F16, bool SEGS, class OUT>
static int vg_start(const VgSide& A, const VgSide& B, const VgArgs& g, cudaStream_t st) {
  CUtensorMap ma, mb;
  if (!vg_map(&ma, A, F16, AMN ? 64 : 128) || !vg_map(&mb, B, F16, BMN ? 64 : BN / 2)) return DELREC_ERR_CUDA;
  auto kern = k_vocab_gemm<BN, AMN, BMN, EPI, F16, SEGS, OUT>;
  SQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)vg_smem(BN)));
  kern<<<kSeqSMs, kVgThreads, vg_smem(BN), st>>>(ma, mb, g);
  SQ_LAUNCHED();
  return DELREC_OK;
}

}  // namespace delrec
