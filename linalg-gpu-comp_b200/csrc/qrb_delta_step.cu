// One token of the gated delta rule per row, for generation (mathematics in qrb_delta.cuh).
//
// A row's state is read once and written once, 8 dk dv bytes that dwarf all else, so memory
// bounds the kernel.  State columns are independent: a block takes 32 of them (128-byte rows, so
// a single row of 16 heads still makes 64 blocks), holds its 16 KB in registers, and reduces
// S~^T k and S~^T q over the rows in one round; o = scale (S~^T q + (k.q) u) then needs no second.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

constexpr int kCols = 32, kStepThreads = 128, kGroups = 16;   // 8 lanes x 4 columns, 16 row groups

template <typename T, bool VEC>
__global__ void __launch_bounds__(kStepThreads) step_kernel(qrb_delta_step_args a, int nt) {
  __shared__ float ks[128], qs[128], part[4][2][kCols], kq_part[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = blockIdx.x % nt, bh = blockIdx.x / nt, h = bh % a.hv, row = bh / a.hv;
  const int hk = h / (a.hv / a.hk);
  const int cl = (tid & 7) * 4, col = tile * kCols + cl, rg = tid >> 3;
  const int slot = a.slots != nullptr ? a.slots[row] : row;
  T* o = static_cast<T*>(a.o) + ((size_t)row * a.hv + h) * a.dv;
  const bool outside = slot < 0 || slot >= a.num_slots;
  // the state rows rg, rg + 16, ...: all loads in flight before anything waits
  float4 s[8];
  const size_t in_slot = ((size_t)h * a.dk) * a.dv + col;
  const float* sp = a.state + (outside ? 0 : (size_t)slot * a.slot_stride + in_slot);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = rg + kGroups * i;
    s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!outside && r < a.dk) {
      if (VEC) {
        if (col < a.dv) s[i] = __ldcs(reinterpret_cast<const float4*>(sp + (size_t)r * a.dv));
      } else {
        const float* x = sp + (size_t)r * a.dv;
        if (col < a.dv) s[i].x = x[0];
        if (col + 1 < a.dv) s[i].y = x[1];
        if (col + 2 < a.dv) s[i].z = x[2];
        if (col + 3 < a.dv) s[i].w = x[3];
      }
    }
  }
  // another, earlier row with this slot?
  int twice = 0;
  if (a.slots != nullptr && !outside)
    for (int j = tid; j < row; j += kStepThreads) twice |= a.slots[j] == slot;
  const T* kp = static_cast<const T*>(a.k) + row * a.k_strides.batch + hk * a.k_strides.head;
  const T* qp = static_cast<const T*>(a.q) + row * a.q_strides.batch + hk * a.q_strides.head;
  ks[tid] = tid < a.dk ? to_f(kp[tid]) : 0.f;
  qs[tid] = tid < a.dk ? to_f(qp[tid]) : 0.f;
  const float kq = warp_sum(ks[tid] * qs[tid]);
  if (lane == 0) kq_part[warp] = kq;
  twice = __syncthreads_or(twice);
  if (outside || twice) {
    if (rg == 0) {
      const T y = from_f<T>(slot < 0 ? 0.f : __int_as_float(0x7fc00000));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < a.dv) o[col + e] = y;
    }
    return;
  }
  const float g = a.g[row * a.g_strides.batch + h * a.g_strides.head];
  const float beta = a.beta[row * a.beta_strides.batch + h * a.beta_strides.head];
  const float decay = expf(g < kMinLog ? kMinLog : g);
  float v[4];
  const T* vp = static_cast<const T*>(a.v) + row * a.v_strides.batch + h * a.v_strides.head;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = col + e < a.dv ? to_f(vp[col + e]) : 0.f;
  float sk[4] = {0.f, 0.f, 0.f, 0.f}, sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float kk = ks[rg + kGroups * i], qq = qs[rg + kGroups * i];
    s[i].x *= decay;
    s[i].y *= decay;
    s[i].z *= decay;
    s[i].w *= decay;
    sk[0] += s[i].x * kk;
    sk[1] += s[i].y * kk;
    sk[2] += s[i].z * kk;
    sk[3] += s[i].w * kk;
    sq[0] += s[i].x * qq;
    sq[1] += s[i].y * qq;
    sq[2] += s[i].z * qq;
    sq[3] += s[i].w * qq;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int off = 8; off < 32; off <<= 1) {
      sk[e] += __shfl_xor_sync(0xffffffffu, sk[e], off);
      sq[e] += __shfl_xor_sync(0xffffffffu, sq[e], off);
    }
    if (lane < 8) {
      part[warp][0][cl + e] = sk[e];
      part[warp][1][cl + e] = sq[e];
    }
  }
  __syncthreads();
  const float kqs = (kq_part[0] + kq_part[1]) + (kq_part[2] + kq_part[3]);
  float u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float k4 = (part[0][0][cl + e] + part[1][0][cl + e]) + (part[2][0][cl + e] + part[3][0][cl + e]);
    const float q4 = (part[0][1][cl + e] + part[1][1][cl + e]) + (part[2][1][cl + e] + part[3][1][cl + e]);
    u[e] = beta * (v[e] - k4);
    if (rg == 0 && col + e < a.dv) o[col + e] = from_f<T>(a.scale * (q4 + kqs * u[e]));
  }
  float* dp = a.state_out + (size_t)slot * a.slot_stride_out + in_slot;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = rg + kGroups * i;
    if (r >= a.dk) continue;
    const float kk = ks[r];
    const float4 y = make_float4(s[i].x + kk * u[0], s[i].y + kk * u[1], s[i].z + kk * u[2], s[i].w + kk * u[3]);
    if (VEC) {
      if (col < a.dv) __stcs(reinterpret_cast<float4*>(dp + (size_t)r * a.dv), y);
    } else {
      float* x = dp + (size_t)r * a.dv;
      if (col < a.dv) x[0] = y.x;
      if (col + 1 < a.dv) x[1] = y.y;
      if (col + 2 < a.dv) x[2] = y.z;
      if (col + 3 < a.dv) x[3] = y.w;
    }
  }
}

template <typename T>
cudaError_t run_step(const qrb_delta_step_args& a, cudaStream_t s) {
  const int nt = (a.dv + kCols - 1) / kCols;
  const bool vec = a.dv % 4 == 0 && a.slot_stride % 4 == 0 && a.slot_stride_out % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.state_out)) & 15u) == 0;
  const double cells = (double)a.batch * a.hv * a.dk * a.dv;
  LaunchTimer t("delta_step_kernel", s, 8.0 * cells, 7.0 * cells);
  const unsigned grid = (unsigned)(a.batch * a.hv * nt);
  if (vec) step_kernel<T, true><<<grid, kStepThreads, 0, s>>>(a, nt);
  else step_kernel<T, false><<<grid, kStepThreads, 0, s>>>(a, nt);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_step(const qrb_delta_step_args& a, cudaStream_t s) {
  if (a.dtype == QRB_BF16) return run_step<__nv_bfloat16>(a, s);
  if (a.dtype == QRB_F16) return run_step<__half>(a, s);
  return run_step<float>(a, s);
}

}  // namespace delta
}  // namespace qrb
