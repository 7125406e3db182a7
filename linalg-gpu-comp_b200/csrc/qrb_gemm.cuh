// Dense products of the linear layer (qrb_gemm.cu), used by qrb_linear.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/qrb200_nn.h"
#include "qrb_internal.cuh"

namespace qrb {
namespace gemm {

// A matrix of `mn` output rows (or columns) by k, bf16 or fp16, 16-byte aligned rows of `ld`
// elements: k along the rows of memory, or with mn_major mn along them.  `pieces` planes of
// `plane` elements each (fp32 operands are three bf16 planes, see split_kernel).
struct Operand {
  const void* p;
  int64_t ld, plane;
  int pieces, mn_major;
};

// What becomes of the product, row m and column n of the output:
//   x = sum + bias[n];  pre[m][n] = x;  y[m][n] = act(x) + residual[m][n].
struct Epilogue {
  int dtype, act;
  void* y;
  int64_t ldy;
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* pre;
  int64_t ldpre;
};

// fp32 scratch elements of multiply() (0 when the product is not split along k).
size_t scratch(int64_t m, int64_t n, int64_t k, int pieces);
// y (m x n) = epilogue(A (m x k) B (n x k)^T).
cudaError_t multiply(const Operand& A, const Operand& B, int64_t m, int64_t n, int64_t k, bool half, const Epilogue& e,
                     float* ws, cudaStream_t s);
int launches(int64_t m, int64_t n, int64_t k, int pieces);
bool supported();   // the driver's tensor map encoder is there

__device__ __forceinline__ float activate(float x, int act) {
  if (act == QRB_ACT_RELU) return x > 0.f ? x : (x != x ? x : 0.f);
  if (act == QRB_ACT_SILU) return x / (1.f + expf(-x));
  if (act == QRB_ACT_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  return x;
}

}  // namespace gemm
}  // namespace qrb
