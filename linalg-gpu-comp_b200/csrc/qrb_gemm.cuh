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
// `plane` elements each (fp32 operands are three bf16 planes, laid out by put8f in qrb_linear.cu).
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
size_t scratch(int64_t m, int64_t n, int64_t k, int pieces, bool half);
// y (m x n) = epilogue(A (m x k) B (n x k)^T).
cudaError_t multiply(const Operand& A, const Operand& B, int64_t m, int64_t n, int64_t k, bool half, const Epilogue& e,
                     float* ws, cudaStream_t s);
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
// Packed fp32 arithmetic: two values an instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// x Phi(x) of two values: phi with s = z sqrt(log2 e) in place of z, q in units of log2 e and with erfc's
// factor 1/2 in it.
__device__ __forceinline__ void gelu2(float& x, float& y) {
  auto both = [](float c) { return pair(c, c); };
  const uint64_t xy = pair(x, y), a = pair(fabsf(x), fabsf(y));
  const uint64_t s = mul2(a, both(8.493218003e-01f)), n = mul2(a, both(-8.493218003e-01f));
  float u, v;
  split(fma2(s, both(4.162773056e-01f), both(1.f)), u, v);
  const uint64_t t = pair(rcp(u), rcp(v));
  uint64_t q = both(2.516222965e-01f);
  q = fma2(q, t, both(-1.210104463e+00f));
  q = fma2(q, t, both(2.194834290e+00f));
  q = fma2(q, t, both(-1.688721258e+00f));
  q = fma2(q, t, both(4.347611031e-01f));
  q = fma2(q, t, both(-2.811356677e-01f));
  q = fma2(q, t, both(1.423633349e-01f));
  q = fma2(q, t, both(5.393846184e-01f));
  q = fma2(q, t, both(1.442744166e+00f));
  q = fma2(q, t, both(-2.825748311e+00f));
  split(fma2(n, s, q), u, v);
  const uint64_t half = mul2(t, pair(ex2(u), ex2(v)));   // erfc(z) / 2
  float h, k;
  split(half, h, k);
  split(fma2(half, both(-1.f), both(1.f)), u, v);
  split(mul2(xy, pair(x < 0.f ? h : u, y < 0.f ? k : v)), x, y);
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
  static_assert(N % 2 == 0, "pairs");
  if (act == QRB_ACT_NONE) return;
  if (act == QRB_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = activate(x[i], QRB_ACT_RELU);
  } else if (act == QRB_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = activate(x[i], QRB_ACT_SILU);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) gelu2(x[i], x[i + 1]);
  }
}

}  // namespace gemm
}  // namespace qrb
