// Products grouped by expert: what the kernels of expert.cu and expert_tc.cu take.
//
// The slots (row * k + choice) stand in the order of their experts; expert e has positions
// [offsets[e], offsets[e + 1]), read on the device, so that no size comes back to the host. Two forms:
//   kRows      C[p] = A[p] B_e^T for each position p of expert e (the forward pass and dx);
//   kWeights   C_e = sum over e's positions of A[p]^T B[p] (dW).
#pragma once

#include "linear.h"

namespace sv {

enum class ExpertForm { kRows, kWeights };

struct ExpertGemm {
  ExpertForm form;
  Operand a;                // kRows: [slots][k]; kWeights: [slots][m], read along m
  Operand b;                // kRows: an expert's [n][k] (or [k][n], mn); kWeights: [slots][n]
  int64_t b_expert;         // kRows: elements between experts' matrices
  const int32_t* offsets;   // [experts + 1]
  int experts;
  int64_t slots;
  int64_t m, n, k;          // kRows: columns n, sum over k; kWeights: an expert's [m][n]
  int dtype;
  bool zero_rest;           // kRows: positions that no expert has are set to zero
  bool runs;                // kRows in fp32: sums over k as near as fp32's own (expert_tc.cu)
  Epilogue ep;              // bias: [experts][n]; out: [slots][n] or [experts][m][n], in out_dtype: dtype,
                            // or fp32 for kRows without zero_rest
};

// expert_tc.cu (fp16 / bf16): operands and strides of multiples of 16 bytes. kWeights needs
// expert_maps_bytes(experts) of workspace, 128-byte aligned.
enum class ExpertTile { kPair256, kPair128, kOne128, kOne64 };
size_t expert_maps_bytes(int experts);
int expert_gemm_tc(const ExpertGemm& g, ExpertTile tile, void* maps, int32_t* status,
                   cudaStream_t s);

}  // namespace sv
