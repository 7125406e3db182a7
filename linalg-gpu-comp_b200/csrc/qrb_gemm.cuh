// Dense products of the linear layer (qrb_gemm.cu), used by qrb_linear.cu.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
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

__device__ __forceinline__ float load1(const void* p, int64_t i, int dtype) {
  if (dtype == QRB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == QRB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store1(void* p, int64_t i, int dtype, float x) {
  if (dtype == QRB_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else if (dtype == QRB_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
  else static_cast<float*>(p)[i] = x;
}

// Phi(x), the normal distribution function, without a branch: with z = |x| / sqrt 2 and
// t = 1 / (1 + z / 2), erfc(z) = t exp(-z^2 + q(t)); q is the degree-9 Chebyshev fit of
// ln(erfc(z) / t) + z^2 on t in [0.05, 1] (below it erfc underflows), computed in 64 bits, within
// 8e-8 of it, 2.2e-7 evaluated in fp32; the exponential adds its argument's rounding.
// (erff takes two paths that a warp walks one after the other, which cost a GELU epilogue 215 cycles
// a value.)
__device__ __forceinline__ float phi(float x) {
  const float z = fabsf(x) * 0.70710678118654752f;
  const float t = __fdividef(1.f, fmaf(0.5f, z, 1.f));
  float q = 1.744112854e-01f;
  q = fmaf(q, t, -8.387804970e-01f);
  q = fmaf(q, t, 1.521343200e+00f);
  q = fmaf(q, t, -1.170532379e+00f);
  q = fmaf(q, t, 3.013534328e-01f);
  q = fmaf(q, t, -1.948683954e-01f);
  q = fmaf(q, t, 9.867874417e-02f);
  q = fmaf(q, t, 3.738729275e-01f);
  q = fmaf(q, t, 1.000034051e+00f);
  q = fmaf(q, t, -1.265512294e+00f);
  const float half = 0.5f * t * __expf(fmaf(-z, z, q));   // erfc(z) / 2
  return x < 0.f ? half : 1.f - half;
}
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

__device__ __forceinline__ float activate(float x, int act) {
  if (act == QRB_ACT_RELU) return x > 0.f ? x : (x != x ? x : 0.f);
  if (act == QRB_ACT_SILU) return x * sigmoid(x);
  if (act == QRB_ACT_GELU) return x * phi(x);
  return x;
}
__device__ __forceinline__ float slope(float x, int act) {
  if (act == QRB_ACT_RELU) return x > 0.f ? 1.f : (x != x ? x : 0.f);
  if (act == QRB_ACT_SILU) {
    const float s = sigmoid(x);
    return s * (1.f + x * (1.f - s));
  }
  if (act == QRB_ACT_GELU) return phi(x) + x * 0.39894228040143268f * __expf(-0.5f * x * x);
  return 1.f;
}

// act over N values at once: one test for all of them.
template <int N>
__device__ __forceinline__ void activate_all(float (&x)[N], int act) {
  if (act == QRB_ACT_NONE) return;
  if (act == QRB_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = activate(x[i], QRB_ACT_RELU);
  } else if (act == QRB_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = activate(x[i], QRB_ACT_SILU);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = activate(x[i], QRB_ACT_GELU);
  }
}

}  // namespace gemm
}  // namespace qrb
