// The linear layer y = act(x w^T + b) + r and its backward pass: C ABI (include/qrb200_nn.h), and
// the elementwise kernels around the products of qrb_gemm.cu.
//
//   forward:  up to four rows: gemv_kernel; otherwise [lay out x, w] product with the epilogue
//   backward: dp = dy act'(pre) and the column sums of dp (dbias), then dx = dp w, dw = dp^T x
// Operands the tensor maps cannot address (rows not 16-byte aligned) are laid out in the workspace
// first, fp32 ones as three bf16 planes.  dp of the 16-bit types is rounded to the type once: it is
// an operand of 16-bit products, whose sums average the roundings out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdarg>
#include <cstdio>

#include "qrb_gemm.cuh"

namespace qrb {
namespace gemm {
namespace {

template <typename T>
__device__ __forceinline__ float tof(T x);
template <>
__device__ __forceinline__ float tof(float x) { return x; }
template <>
__device__ __forceinline__ float tof(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float tof(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T fromf(float x);
template <>
__device__ __forceinline__ float fromf(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 fromf(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half fromf(float x) { return __float2half_rn(x); }

// Eight neighbouring values of a laid-out operand (those behind `count` become zero): the values
// themselves, or the three bf16 planes of fp32 ones.  A value that is not finite keeps its first plane
// only (inf - inf would put NaN into the others).
template <typename T>
__device__ __forceinline__ void put8f(void* to, int64_t i, int64_t plane, const float (&e)[8], int count) {
  constexpr int P = sizeof(T) == 4 ? 3 : 1;
  uint32_t w[P][4];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    if (P == 1) {
      T pair[2] = {fromf<T>(j < count ? e[j] : 0.f), fromf<T>(j + 1 < count ? e[j + 1] : 0.f)};
      w[0][j / 2] = *reinterpret_cast<const uint32_t*>(pair);
    } else {
      __align__(4) __nv_bfloat16 pc[3][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = j + h < count ? e[j + h] : 0.f;
        pc[0][h] = __float2bfloat16_rn(x);
        // the last half step below fp32's largest value would round to infinity: down, the rest follows
        if (__hisinf(pc[0][h]) && fabsf(x) <= 3.402823466e38f) pc[0][h] = __float2bfloat16_rz(x);
        float r = x - __bfloat162float(pc[0][h]);
        if (!(fabsf(r) <= 3.4e38f)) r = 0.f;
        pc[1][h] = __float2bfloat16_rn(r);
        pc[2][h] = __float2bfloat16_rn(r - __bfloat162float(pc[1][h]));
      }
#pragma unroll
      for (int q = 0; q < P; ++q) w[q][j / 2] = *reinterpret_cast<const uint32_t*>(pc[q]);
    }
  }
#pragma unroll
  for (int q = 0; q < P; ++q)
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(to) + i + q * plane) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
}

// rows x cols of `from` (row stride ld) to rows of `pitch` elements: eight columns a thread, stored as
// 16-byte units (the columns that pad a row become zero).  Up to two matrices a launch (blockIdx.z).
template <typename T>
struct LayoutJob {
  const T* from;
  int64_t ld, rows, cols, pitch;
  void* to;
};
template <typename T>
__global__ void __launch_bounds__(256) layout_kernel(LayoutJob<T> a, LayoutJob<T> b) {
  const LayoutJob<T>& g = blockIdx.z == 0 ? a : b;
  const int64_t c = ((int64_t)blockIdx.x * 32 + (threadIdx.x & 31)) * 8, plane = g.rows * g.pitch;
  if (c >= g.pitch) return;
  for (int64_t r = (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5); r < g.rows; r += (int64_t)gridDim.y * 8) {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = tof(__ldg(g.from + r * g.ld + min(c + j, g.cols - 1)));
    put8f<T>(g.to, r * g.pitch + c, plane, e, (int)min((int64_t)8, g.cols - c));
  }
}

constexpr int kSumRows = 64, kSumCols = 256;   // rows and columns a block of dp_kernel covers

// Eight neighbouring values; VEC: one or two 16-byte loads, otherwise existing columns only.
template <typename T, bool VEC>
__device__ __forceinline__ void get8(const T* p, int count, T (&e)[8]) {
  if (VEC) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j)
      reinterpret_cast<uint4*>(e)[j] = __ldg(reinterpret_cast<const uint4*>(p) + j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = __ldg(p + min(j, count - 1));
  }
}

// dp = dy act'(pre) into a laid-out operand (to, unless null) and its column sums over the block's
// rows (sums[row block][n], unless null).  Sums are of the fp32 products, before any rounding.  A
// thread takes eight columns of every eighth row, four rows in flight.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dp_kernel(const T* dy, int64_t ldy, const T* pre, int64_t ldp, int act,
                                                 int64_t m, int64_t n, void* to, int64_t pitch, float* sums) {
  __shared__ float part[8][kSumCols];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * kSumCols + 8 * lane, r0 = (int64_t)blockIdx.y * kSumRows;
  const int count = (int)min((int64_t)8, n - col);
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = 0.f;
  if (count > 0) {
    for (int i = g; i < kSumRows; i += 32) {
      alignas(16) T a[4][8], b[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t r = min(r0 + i + 8 * u, m - 1);
        get8<T, VEC>(dy + r * ldy + col, count, a[u]);
        if (act != QRB_ACT_NONE) get8<T, VEC>(pre + r * ldp + col, count, b[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t r = r0 + i + 8 * u;
        if (r >= m) continue;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = tof(a[u][j]);
          if (act != QRB_ACT_NONE) x[j] *= slope(tof(b[u][j]), act);
          s[j] += x[j];
        }
        if (to != nullptr) put8f<T>(to, r * pitch + col, m * pitch, x, count);
      }
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) part[g][8 * lane + j] = s[j];
  __syncthreads();
  const int c = threadIdx.x;
  if ((int64_t)blockIdx.x * kSumCols + c < n) {
    float t = part[0][c];
#pragma unroll
    for (int i = 1; i < 8; ++i) t += part[i][c];
    sums[(int64_t)blockIdx.y * n + (int64_t)blockIdx.x * kSumCols + c] = t;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(const float* sums, int64_t blocks, int64_t n, T* out) {
  __shared__ float part[8][32];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < n)
    for (int64_t b = g; b < blocks; b += 8) s += sums[b * n + col];
  part[g][c] = s;
  __syncthreads();
  if (g == 0 && col < n) {
    for (int i = 1; i < 8; ++i) s += part[i][c];
    out[col] = fromf<T>(s);
  }
}

// y = epilogue(x w^T) for up to four rows, which the weight's bytes bound: a warp (SPLIT: the eight
// warps of a block, for outputs too few to fill the card with warps) takes one row of w, 16 bytes a
// lane and eight loads in flight; x comes from L1.  fp32 sums in a fixed order.
template <typename T, int M, bool VEC, bool SPLIT>
__global__ void __launch_bounds__(256) gemv_kernel(const T* x, int64_t ldx, const T* w, int64_t ldw, int64_t k, int64_t n,
                                                   Epilogue e) {
  constexpr int V = 16 / (int)sizeof(T), U = 8;   // elements a lane takes at once, times in flight
  __shared__ float part[8][M];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = SPLIT ? blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
  if (!SPLIT && c >= n) return;
  const T* wr = w + c * ldw;
  float s[M];
#pragma unroll
  for (int i = 0; i < M; ++i) s[i] = 0.f;
  const int64_t step = (SPLIT ? 8 : 1) * 32 * V, begin = (SPLIT ? threadIdx.x : lane) * V;
  // the same elements to the same lane whatever the alignment: results do not depend on it
  auto get = [&](T (&to)[V], const T* from, int64_t at) {
    if (VEC) {
      *reinterpret_cast<uint4*>(to) = __ldg(reinterpret_cast<const uint4*>(from + at));
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) to[j] = __ldg(from + min(at + j, k - 1));
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j >= k) to[j] = fromf<T>(0.f);
    }
  };
  auto use = [&](const T (&we)[V], int64_t at) {
#pragma unroll
    for (int i = 0; i < M; ++i) {
      alignas(16) T xe[V];
      get(xe, x + i * ldx, at);
#pragma unroll
      for (int j = 0; j < V; ++j) s[i] = fmaf(tof(we[j]), tof(xe[j]), s[i]);
    }
  };
  int64_t at = begin;
  for (; at + (U - 1) * step < k; at += U * step) {
    alignas(16) T we[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) get(we[u], wr, at + u * step);
#pragma unroll
    for (int u = 0; u < U; ++u) use(we[u], at + u * step);
  }
  for (; at < k; at += step) {
    alignas(16) T we[V];
    get(we, wr, at);
    use(we, at);
  }
#pragma unroll
  for (int i = 0; i < M; ++i) s[i] = warp_sum(s[i]);
  if (SPLIT) {
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < M; ++i) part[warp][i] = s[i];
    __syncthreads();
    if (threadIdx.x >= M) return;
#pragma unroll
    for (int i = 0; i < M; ++i)
      if (i == (int)threadIdx.x) {
        s[0] = part[0][i];
        for (int j = 1; j < 8; ++j) s[0] += part[j][i];
      }
  } else {
#pragma unroll
    for (int i = 1; i < M; ++i)
      if (lane == i) s[0] = s[i];
    if (lane >= M) return;
  }
  const int64_t r = SPLIT ? threadIdx.x : lane;   // lane r finishes row r
  float v = s[0] + (e.bias != nullptr ? load1(e.bias, c, e.dtype) : 0.f);
  if (e.pre != nullptr) store1(e.pre, r * e.ldpre + c, e.dtype, v);
  v = activate(v, e.act);
  if (e.residual != nullptr) v += load1(e.residual, r * e.ldr + c, e.dtype);
  store1(e.y, r * e.ldy + c, e.dtype, v);
}

}  // namespace
}  // namespace gemm
}  // namespace qrb

namespace {

using qrb::gemm::Epilogue;
using qrb::gemm::Operand;

int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return qrb::set_error(status, buf);
}

#define TRY(x)                   \
  do {                           \
    int _s = (x);                \
    if (_s != QRB_OK) return _s; \
  } while (0)
#define CUDA(x, what)                                                                               \
  do {                                                                                              \
    cudaError_t _e = (x);                                                                           \
    if (_e != cudaSuccess)                                                                          \
      return fail(QRB_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(_e), cudaGetErrorString(_e)); \
  } while (0)

size_t al(size_t x) { return (x + 255) & ~size_t(255); }
size_t esize(int dtype) { return dtype == QRB_F32 ? 4 : 2; }
int64_t pitch_of(int64_t cols) { return (cols + 7) / 8 * 8; }

// Whether the tensor maps can read the rows as they lie.
bool direct(int dtype, const void* p, int64_t ld, int64_t cols) {
  return dtype != QRB_F32 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0 && ld >= cols;
}
size_t layout_bytes(int dtype, int64_t rows, int64_t cols) {
  return al((size_t)rows * pitch_of(cols) * 2 * (dtype == QRB_F32 ? 3 : 1));
}

int check_common(int dtype, int act, int64_t m, int64_t k, int64_t n) {
  if (dtype != QRB_F32 && dtype != QRB_BF16 && dtype != QRB_F16)
    return fail(QRB_ERR_INVALID_ARG, "dtype must be QRB_F32, QRB_BF16 or QRB_F16 (got %d)", dtype);
  if (act < QRB_ACT_NONE || act > QRB_ACT_GELU) return fail(QRB_ERR_INVALID_ARG, "unknown activation %d", act);
  if (m < 0 || n < 1 || k < 1)
    return fail(QRB_ERR_INVALID_ARG, "m must be >= 0, k and n >= 1 (got %lld, %lld, %lld)", (long long)m, (long long)k,
                (long long)n);
  const int64_t top = (int64_t)1 << 30;
  if (m > top || n > top || k > top || (m > 0 && m * n / (128 * 64) > top / 16) || k * n / (128 * 64) > top / 16 ||
      m * k / (128 * 64) > top / 16 || m > (int64_t)64 * 65535)
    return fail(QRB_ERR_UNSUPPORTED, "sizes m = %lld, k = %lld, n = %lld are too large", (long long)m, (long long)k,
                (long long)n);
  return QRB_OK;
}

int check_ptr(const void* p, const char* name, int dtype) {
  if (p == nullptr) return fail(QRB_ERR_INVALID_ARG, "%s is null", name);
  if ((reinterpret_cast<uintptr_t>(p) & (esize(dtype) - 1)) != 0)
    return fail(QRB_ERR_INVALID_ARG, "%s must be %zu-byte aligned", name, esize(dtype));
  return QRB_OK;
}

int check_ld(int64_t ld, int64_t cols, const char* name) {
  if (ld < cols) return fail(QRB_ERR_INVALID_ARG, "%s must be at least %lld (got %lld)", name, (long long)cols, (long long)ld);
  return QRB_OK;
}

int check_device() {
  int dev = 0, major = 0;
  CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  static int cache[64] = {0};
  if (dev < 64) major = cache[dev];
  if (major == 0) {
    CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev), "cudaDeviceGetAttribute");
    if (dev < 64) cache[dev] = major;
  }
  if (major != 10)
    return fail(QRB_ERR_DEVICE, "device %d has compute capability %d.x; libqrb200 needs sm_100", dev, major);
  if (!qrb::gemm::supported()) return fail(QRB_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
  return QRB_OK;
}

int check_ws(const void* ws, size_t have, size_t need) {
  if (need > 0 && (ws == nullptr || have < need))
    return fail(QRB_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given%s", need, have,
                ws == nullptr ? " (null)" : "");
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & 255u) != 0)
    return fail(QRB_ERR_INVALID_ARG, "workspace must be 256-byte aligned");
  return QRB_OK;
}

// The operands a product reads: x (rows x cols, row stride ld) itself, or a copy that a Layouts call makes.
struct Layouts {
  int dtype;
  struct Job {
    const void* p;
    int64_t ld, rows, cols;
    void* to;
  } job[2];
  int jobs = 0;

  explicit Layouts(int dtype_) : dtype(dtype_) {}

  Operand operand(const void* p, int64_t ld, int64_t rows, int64_t cols, bool mn_major, void* to) {
    Operand o{};
    o.mn_major = mn_major;
    o.pieces = dtype == QRB_F32 ? 3 : 1;
    if (direct(dtype, p, ld, cols)) {
      o.p = p;
      o.ld = ld;
      return o;
    }
    o.p = to;
    o.ld = pitch_of(cols);
    o.plane = rows * o.ld;
    job[jobs++] = {p, ld, rows, cols, to};
    return o;
  }

  template <typename T>
  void go(cudaStream_t s) const {
    qrb::gemm::LayoutJob<T> j[2]{};
    int64_t px = 0, py = 0;
    for (int i = 0; i < jobs; ++i) {
      j[i] = {static_cast<const T*>(job[i].p), job[i].ld, job[i].rows, job[i].cols, pitch_of(job[i].cols), job[i].to};
      if (j[i].pitch > px) px = j[i].pitch;
      if (j[i].rows > py) py = j[i].rows;
    }
    py = (py + 7) / 8;
    const dim3 grid((unsigned)((px + 255) / 256), (unsigned)(py < 4096 ? py : 4096), (unsigned)jobs);
    qrb::gemm::layout_kernel<T><<<grid, 256, 0, s>>>(j[0], j[1]);
  }

  int run(cudaStream_t s) const {
    if (jobs == 0) return QRB_OK;
    double cells = 0;
    for (int i = 0; i < jobs; ++i) cells += (double)job[i].rows * job[i].cols;
    qrb::LaunchTimer t("linear_layout_kernel", s, cells * (dtype == QRB_F32 ? 10 : 4), 0);
    if (dtype == QRB_F32) go<float>(s);
    else if (dtype == QRB_BF16) go<__nv_bfloat16>(s);
    else go<__half>(s);
    CUDA(cudaGetLastError(), "linear layout launch");
    return QRB_OK;
  }
};

constexpr int64_t kVecRows = 4;   // up to here gemv_kernel: it reads the weight once and lays nothing out

template <typename T, int M>
cudaError_t run_gemv(const qrb_linear_args& a, const Epilogue& e, cudaStream_t s) {
  const int64_t v = 16 / (int64_t)sizeof(T);
  const bool vec = a.k % v == 0 && a.ldx % v == 0 && a.ldw % v == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w)) & 15u) == 0;
  // eight warps a column where a warp each would leave most of the card without one
  const bool split = a.n < 4 * (int64_t)qrb::sm_count() && a.k >= 1024;
  const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.w);
  const unsigned grid = (unsigned)(split ? a.n : (a.n + 7) / 8);
  qrb::LaunchTimer t("linear_gemv_kernel", s, (double)(a.m + a.n) * a.k * sizeof(T), 2.0 * a.m * a.n * a.k);
  using namespace qrb::gemm;
  if (vec) {
    if (split) gemv_kernel<T, M, true, true><<<grid, 256, 0, s>>>(x, a.ldx, w, a.ldw, a.k, a.n, e);
    else gemv_kernel<T, M, true, false><<<grid, 256, 0, s>>>(x, a.ldx, w, a.ldw, a.k, a.n, e);
  } else {
    if (split) gemv_kernel<T, M, false, true><<<grid, 256, 0, s>>>(x, a.ldx, w, a.ldw, a.k, a.n, e);
    else gemv_kernel<T, M, false, false><<<grid, 256, 0, s>>>(x, a.ldx, w, a.ldw, a.k, a.n, e);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t pick_gemv(const qrb_linear_args& a, const Epilogue& e, cudaStream_t s) {
  switch (a.m) {
    case 1: return run_gemv<T, 1>(a, e, s);
    case 2: return run_gemv<T, 2>(a, e, s);
    case 3: return run_gemv<T, 3>(a, e, s);
    default: return run_gemv<T, 4>(a, e, s);
  }
}

struct FwdLayout {
  size_t x, w, part, total;
};
FwdLayout fwd_layout(const qrb_linear_args& a) {
  FwdLayout l{};
  if (a.m <= kVecRows) return l;
  size_t at = 0;
  l.x = at;
  if (!direct(a.dtype, a.x, a.ldx, a.k)) at += layout_bytes(a.dtype, a.m, a.k);
  l.w = at;
  if (!direct(a.dtype, a.w, a.ldw, a.k)) at += layout_bytes(a.dtype, a.n, a.k);
  l.part = at;
  at += al(qrb::gemm::scratch(a.m, a.n, a.k, a.dtype == QRB_F32 ? 3 : 1, a.dtype == QRB_F16) * 4);
  l.total = at;
  return l;
}

int check_forward(const qrb_linear_args* a) {
  if (a == nullptr) return fail(QRB_ERR_INVALID_ARG, "args is null");
  TRY(check_common(a->dtype, a->activation, a->m, a->k, a->n));
  TRY(check_ld(a->ldx, a->k, "ldx"));
  TRY(check_ld(a->ldw, a->k, "ldw"));
  return QRB_OK;
}

struct BwdLayout {
  size_t dp, x, w, sums, part, total;
};
bool makes_dp(const qrb_linear_backward_args& a) {
  return a.activation != QRB_ACT_NONE || !direct(a.dtype, a.dy, a.lddy, a.n);
}
BwdLayout bwd_layout(const qrb_linear_backward_args& a) {
  const int pieces = a.dtype == QRB_F32 ? 3 : 1;
  BwdLayout l{};
  size_t at = 0;
  l.dp = at;
  if (makes_dp(a)) at += layout_bytes(a.dtype, a.m, a.n);
  l.x = at;
  if (!direct(a.dtype, a.x, a.ldx, a.k)) at += layout_bytes(a.dtype, a.m, a.k);
  l.w = at;
  if (!direct(a.dtype, a.w, a.ldw, a.k)) at += layout_bytes(a.dtype, a.n, a.k);
  l.sums = at;
  at += al((size_t)((a.m + qrb::gemm::kSumRows - 1) / qrb::gemm::kSumRows) * a.n * 4);
  l.part = at;
  const bool half = a.dtype == QRB_F16;
  const size_t p1 = qrb::gemm::scratch(a.m, a.k, a.n, pieces, half), p2 = qrb::gemm::scratch(a.n, a.k, a.m, pieces, half);
  at += al((p1 > p2 ? p1 : p2) * 4);
  l.total = at;
  return l;
}

int check_backward(const qrb_linear_backward_args* a) {
  if (a == nullptr) return fail(QRB_ERR_INVALID_ARG, "args is null");
  TRY(check_common(a->dtype, a->activation, a->m, a->k, a->n));
  TRY(check_ld(a->lddy, a->n, "lddy"));
  TRY(check_ld(a->ldx, a->k, "ldx"));
  TRY(check_ld(a->ldw, a->k, "ldw"));
  if (a->activation != QRB_ACT_NONE) TRY(check_ld(a->ldpre, a->n, "ldpre"));
  return QRB_OK;
}

template <typename T>
int run_dp(const qrb_linear_backward_args& a, void* to, float* sums, cudaStream_t s) {
  const int64_t rb = (a.m + qrb::gemm::kSumRows - 1) / qrb::gemm::kSumRows;
  {
    qrb::LaunchTimer t("linear_dp_kernel", s, (double)a.m * a.n * sizeof(T) * 3, (double)a.m * a.n);
    const dim3 grid((unsigned)((a.n + qrb::gemm::kSumCols - 1) / qrb::gemm::kSumCols), (unsigned)rb);
    const int64_t v = 16 / (int64_t)sizeof(T);
    const bool vec = a.n % 8 == 0 && a.lddy % v == 0 && (reinterpret_cast<uintptr_t>(a.dy) & 15u) == 0 &&
                     (a.activation == QRB_ACT_NONE ||
                      (a.ldpre % v == 0 && (reinterpret_cast<uintptr_t>(a.pre) & 15u) == 0));
    auto kernel = vec ? qrb::gemm::dp_kernel<T, true> : qrb::gemm::dp_kernel<T, false>;
    kernel<<<grid, 256, 0, s>>>(static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.pre), a.ldpre, a.activation,
                                a.m, a.n, to, pitch_of(a.n), sums);
    CUDA(cudaGetLastError(), "linear dp launch");
  }
  if (sums != nullptr) {
    qrb::LaunchTimer t("linear_colsum_kernel", s, 4.0 * rb * a.n, (double)rb * a.n);
    qrb::gemm::colsum_kernel<T><<<(unsigned)((a.n + 31) / 32), 256, 0, s>>>(sums, rb, a.n, static_cast<T*>(a.dbias));
    CUDA(cudaGetLastError(), "linear column sum launch");
  }
  return QRB_OK;
}

}  // namespace

extern "C" {

size_t qrb_linear_workspace_size(const qrb_linear_args* a) {
  if (check_forward(a) != QRB_OK || a->m == 0) return 0;
  return fwd_layout(*a).total;
}

int qrb_linear_forward(const qrb_linear_args* a, void* ws, size_t wsb, void* stream) {
  TRY(check_forward(a));
  if (a->m == 0) return QRB_OK;
  TRY(check_ptr(a->x, "x", a->dtype));
  TRY(check_ptr(a->w, "w", a->dtype));
  TRY(check_ptr(a->y, "y", a->dtype));
  TRY(check_ld(a->ldy, a->n, "ldy"));
  if (a->bias != nullptr) TRY(check_ptr(a->bias, "bias", a->dtype));
  if (a->residual != nullptr) {
    TRY(check_ptr(a->residual, "residual", a->dtype));
    TRY(check_ld(a->ldr, a->n, "ldr"));
  }
  if (a->pre != nullptr) {
    TRY(check_ptr(a->pre, "pre", a->dtype));
    TRY(check_ld(a->ldpre, a->n, "ldpre"));
  }
  const FwdLayout l = fwd_layout(*a);
  TRY(check_ws(ws, wsb, l.total));
  TRY(check_device());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Epilogue e{a->dtype, a->activation, a->y, a->ldy, a->bias, a->residual, a->ldr, a->pre, a->ldpre};
  if (a->m <= kVecRows) {
    CUDA(a->dtype == QRB_F32    ? pick_gemv<float>(*a, e, s)
         : a->dtype == QRB_BF16 ? pick_gemv<__nv_bfloat16>(*a, e, s)
                                : pick_gemv<__half>(*a, e, s),
         "linear few-row launch");
    return QRB_OK;
  }
  char* w8 = static_cast<char*>(ws);
  Layouts lay(a->dtype);
  const Operand x = lay.operand(a->x, a->ldx, a->m, a->k, false, w8 + l.x);
  const Operand w = lay.operand(a->w, a->ldw, a->n, a->k, false, w8 + l.w);
  TRY(lay.run(s));
  CUDA(qrb::gemm::multiply(x, w, a->m, a->n, a->k, a->dtype == QRB_F16, e, reinterpret_cast<float*>(w8 + l.part), s),
       "linear product launch");
  return QRB_OK;
}

size_t qrb_linear_backward_workspace_size(const qrb_linear_backward_args* a) {
  if (check_backward(a) != QRB_OK || a->m == 0) return 0;
  return bwd_layout(*a).total;
}

int qrb_linear_backward(const qrb_linear_backward_args* a, void* ws, size_t wsb, void* stream) {
  TRY(check_backward(a));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t es = esize(a->dtype);
  if (a->dw != nullptr) TRY(check_ptr(a->dw, "dw", a->dtype));
  if (a->dbias != nullptr) TRY(check_ptr(a->dbias, "dbias", a->dtype));
  if (a->m == 0) {   // sums over no rows
    if (a->dw != nullptr) CUDA(cudaMemsetAsync(a->dw, 0, (size_t)a->n * a->k * es, s), "dw = 0");
    if (a->dbias != nullptr) CUDA(cudaMemsetAsync(a->dbias, 0, (size_t)a->n * es, s), "dbias = 0");
    return QRB_OK;
  }
  TRY(check_ptr(a->dy, "dy", a->dtype));
  if (a->activation != QRB_ACT_NONE) TRY(check_ptr(a->pre, "pre", a->dtype));
  if (a->dw != nullptr) TRY(check_ptr(a->x, "x", a->dtype));
  if (a->dx != nullptr) {
    TRY(check_ptr(a->w, "w", a->dtype));
    TRY(check_ptr(a->dx, "dx", a->dtype));
  }
  const BwdLayout l = bwd_layout(*a);
  TRY(check_ws(ws, wsb, l.total));
  TRY(check_device());
  char* w8 = static_cast<char*>(ws);
  const bool half = a->dtype == QRB_F16, dp = makes_dp(*a) && (a->dx != nullptr || a->dw != nullptr);
  float* sums = a->dbias != nullptr ? reinterpret_cast<float*>(w8 + l.sums) : nullptr;
  if (dp || sums != nullptr) {
    void* to = dp ? w8 + l.dp : nullptr;
    if (a->dtype == QRB_F32) TRY(run_dp<float>(*a, to, sums, s));
    else if (half) TRY(run_dp<__half>(*a, to, sums, s));
    else TRY(run_dp<__nv_bfloat16>(*a, to, sums, s));
  }
  Operand p{};
  p.pieces = a->dtype == QRB_F32 ? 3 : 1;
  if (makes_dp(*a)) {
    p.p = w8 + l.dp;
    p.ld = pitch_of(a->n);
    p.plane = a->m * p.ld;
  } else {
    p.p = a->dy;
    p.ld = a->lddy;
  }
  float* part = reinterpret_cast<float*>(w8 + l.part);
  Epilogue e{};
  e.dtype = a->dtype;
  e.ldy = a->k;
  Layouts lay(a->dtype);
  Operand x{}, w{};
  if (a->dx != nullptr) w = lay.operand(a->w, a->ldw, a->n, a->k, true, w8 + l.w);
  if (a->dw != nullptr) x = lay.operand(a->x, a->ldx, a->m, a->k, true, w8 + l.x);
  TRY(lay.run(s));
  if (a->dx != nullptr) {
    p.mn_major = 0;
    e.y = a->dx;
    CUDA(qrb::gemm::multiply(p, w, a->m, a->k, a->n, half, e, part, s), "linear dx launch");
  }
  if (a->dw != nullptr) {
    p.mn_major = 1;
    e.y = a->dw;
    CUDA(qrb::gemm::multiply(p, x, a->n, a->k, a->m, half, e, part, s), "linear dw launch");
  }
  return QRB_OK;
}

}  // extern "C"
