// Per-chunk factors of the gated delta rule (mathematics in qrb_delta.cuh).
//
//   plan_kernel  packed layout: first chunk slot of every sequence (one block, a prefix sum).
//   prep_kernel  one block per (chunk, value head): the running decays, X and P of the chunk,
//                and the chunk's q, k, v (and dO) as zero-padded tiles.  These depend on no state,
//                so all chunks run at once and the sequential kernels are left with products only.
//
// X is solved column by column in fp32: thread j owns column j, the rows of M are broadcast
// from shared memory, 2016 multiply-adds a thread in four independent sums.  It is a T factor's
// recurrence, bound by issue, and blocks of other chunks fill the SM beside it.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

__global__ void __launch_bounds__(1024) plan_kernel(Params p) {
  __shared__ int part[1024];
  const int tid = threadIdx.x;
  const int per = (p.nseq + 1023) / 1024;
  int64_t sum = 0;
  for (int i = 0; i < per; ++i) {
    const int s = tid * per + i;
    if (s < p.nseq) {
      int64_t b, t0, n;
      seq_range(p, s, b, t0, n);
      sum += (n + kChunk - 1) / kChunk;
    }
  }
  part[tid] = (int)(sum < p.bound ? sum : p.bound);
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    int64_t v = part[tid];
    if (tid >= o) v += part[tid - o];
    __syncthreads();
    part[tid] = (int)(v < p.bound ? v : p.bound);
    __syncthreads();
  }
  int64_t at = tid == 0 ? 0 : part[tid - 1];
  for (int i = 0; i < per; ++i) {
    const int s = tid * per + i;
    if (s < p.nseq) {
      p.cstart[s] = (int)at;
      int64_t b, t0, n;
      seq_range(p, s, b, t0, n);
      at += (n + kChunk - 1) / kChunk;
      if (at > p.bound) at = p.bound;
      if (s == p.nseq - 1) p.cstart[p.nseq] = (int)at;
    }
  }
}

template <int DKP, typename T, int PS>
constexpr int prep_operands() {
  constexpr int qk = 2 * tile_bytes(kChunk, Pieces<T>::kIn, DKP);
  constexpr int xp = 2 * tile_bytes(kChunk, PS, kChunk);
  return qk > xp ? qk : xp;
}
constexpr int kMStride = 68;   // floats per row of M: rows stay 16-byte aligned, columns on distinct banks

template <int DKP, typename T, int PS>
constexpr int prep_smem() {
  return prep_operands<DKP, T, PS>() + kChunk * kMStride * 4 + kChunk * 8 + kChunk * 4;
}

// Rows of x (dense last dimension of d <= DKP) as zero-padded pieces.
template <int DKP, typename T>
__device__ void load_rows(unsigned char* tile, const T* x, int64_t row_stride, int len, int d, bool vec) {
  constexpr int P = Pieces<T>::kIn;
  constexpr int V = 16 / sizeof(T);
  if (vec) {
    for (int u = threadIdx.x; u < kChunk * (DKP / V); u += blockDim.x) {
      const int r = u / (DKP / V), c = (u % (DKP / V)) * V;
      alignas(16) T e[V];
      if (r < len && c < d)
        *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(x + r * row_stride + c);
      else
        *reinterpret_cast<uint4*>(e) = make_uint4(0, 0, 0, 0);
      if (P == 1) {
        *reinterpret_cast<uint4*>(tile + tile_off(kChunk, r, c)) = *reinterpret_cast<uint4*>(e);
      } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) put2<P>(tile, kChunk, DKP, r, c + i, to_f(e[i]), to_f(e[i + 1]));
      }
    }
    return;
  }
  for (int u = threadIdx.x; u < kChunk * (DKP / 2); u += blockDim.x) {
    const int r = u / (DKP / 2), c = (u % (DKP / 2)) * 2;
    const float a = r < len && c < d ? to_f(x[r * row_stride + c]) : 0.f;
    const float b = r < len && c + 1 < d ? to_f(x[r * row_stride + c + 1]) : 0.f;
    put2<P>(tile, kChunk, DKP, r, c, a, b);
  }
}

// v or dO of the chunk as kChunk x 128 tiles (one per 128 value columns), zero-padded: what the
// recurrences then read needs no test of rows, columns or alignment.
template <typename T>
__device__ void stage_rows(unsigned char* to, const T* x, int64_t row_stride, int len, int dv, bool vec) {
  constexpr int V = 16 / sizeof(T);
  const int nb = (dv + 127) / 128;
  for (int u = threadIdx.x; u < nb * kChunk * (128 / V); u += blockDim.x) {
    const int r = (u / (128 / V)) % kChunk, c = (u % (128 / V)) * V, col = u / (kChunk * 128 / V) * 128 + c;
    alignas(16) T e[V];
    if (r < len && vec && col + V <= dv) {
      *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(x + r * row_stride + col);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = r < len && col + i < dv ? x[r * row_stride + col + i] : from_f<T>(0.f);
    }
    *reinterpret_cast<uint4*>(to + (size_t)u * 16) = *reinterpret_cast<uint4*>(e);
  }
}

template <typename T>
__device__ void zero_rows(const Params& p, int idx, int h) {
  int64_t end = p.offsets[p.nseq];
  end = end < 0 ? 0 : end;
  const int64_t t0 = end + (int64_t)idx * kChunk;
  for (int r = 0; r < kChunk; ++r) {
    const int64_t t = t0 + r;
    if (t >= p.time) return;
    if (!p.backward) {
      T* o = static_cast<T*>(p.o) + t * p.os.t + h * p.os.h;
      for (int c = threadIdx.x; c < p.dv; c += blockDim.x) o[c] = from_f<T>(0.f);
    } else {
      T* dv = static_cast<T*>(p.dv_) + (t * p.hv + h) * p.dv;
      for (int c = threadIdx.x; c < p.dv; c += blockDim.x) dv[c] = from_f<T>(0.f);
      if (h < p.hk) {
        T* dq = static_cast<T*>(p.dq) + (t * p.hk + h) * p.dk;
        T* dk = static_cast<T*>(p.dk_) + (t * p.hk + h) * p.dk;
        for (int c = threadIdx.x; c < p.dk; c += blockDim.x) dq[c] = dk[c] = from_f<T>(0.f);
      }
      if (threadIdx.x == 0) p.dg[t * p.hv + h] = p.dbeta[t * p.hv + h] = 0.f;
    }
  }
}

template <int DKP, typename T, int PS>
__global__ void __launch_bounds__(128) prep_kernel(Params p, int vec) {
  constexpr int P = Pieces<T>::kIn;
  constexpr int kQK = tile_bytes(kChunk, P, DKP), kXP = tile_bytes(kChunk, PS, kChunk);
  extern __shared__ __align__(128) unsigned char sm[];
  unsigned char *kt = sm, *qt = sm + kQK, *xt = sm, *pt = sm + kXP;
  float* M = reinterpret_cast<float*>(sm + prep_operands<DKP, T, PS>());
  double* G = reinterpret_cast<double*>(M + kChunk * kMStride);
  float* beta = reinterpret_cast<float*>(G + kChunk);
  const int c = blockIdx.x, h = blockIdx.y, hk = h / p.group, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Chunk ch = chunk_at(p, c);
  if (ch.seq < 0) {
    if (p.zero_tail) zero_rows<T>(p, ch.idx, h);
    return;
  }
  load_rows<DKP, T>(kt, static_cast<const T*>(p.k) + ch.b * p.ks.b + ch.t0 * p.ks.t + hk * p.ks.h, p.ks.t, ch.len,
                    p.dk, vec & 1);
  load_rows<DKP, T>(qt, static_cast<const T*>(p.q) + ch.b * p.qs.b + ch.t0 * p.qs.t + hk * p.qs.h, p.qs.t, ch.len,
                    p.dk, vec & 2);
  const size_t sh = slot_head(p, c, h);
  const size_t vat = sh * ((p.dv + 127) / 128) * kChunk * 128 * sizeof(T);
  stage_rows<T>(p.vt + vat, static_cast<const T*>(p.v) + ch.b * p.vs.b + ch.t0 * p.vs.t + h * p.vs.h, p.vs.t, ch.len,
                p.dv, vec & 4);
  if (p.backward)
    stage_rows<T>(p.dot + vat, static_cast<const T*>(p.d_o) + ch.b * p.dos.b + ch.t0 * p.dos.t + h * p.dos.h, p.dos.t,
                  ch.len, p.dv, vec & 8);
  if (warp == 0) {
    // Running sums of g in fp64: differences of far apart sums keep their low bits.
    const int64_t gbase = ch.b * p.gs.b + ch.t0 * p.gs.t + h * p.gs.h;
    const int64_t bbase = ch.b * p.bs.b + ch.t0 * p.bs.t + h * p.bs.h;
    double g[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * lane + e;
      float x = 0.f, b = 0.f;
      if (i < ch.len) {
        x = p.g[gbase + i * p.gs.t];
        b = p.beta[bbase + i * p.bs.t];
        if (x < kMinLog) x = kMinLog;
      }
      g[e] = x;
      beta[i] = b;
    }
    double s = g[0] + g[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const double last = __shfl_sync(0xffffffffu, s, 31);
    const double g1 = s, g0 = s - g[1];
    G[2 * lane] = g0;
    G[2 * lane + 1] = g1;
    float* gt = p.gates + sh * 3 * kChunk;
    gt[2 * lane] = expf((float)g0);
    gt[2 * lane + 1] = expf((float)g1);
    gt[kChunk + 2 * lane] = expf((float)(last - g0));
    gt[kChunk + 2 * lane + 1] = expf((float)(last - g1));
    gt[2 * kChunk + 2 * lane] = beta[2 * lane];
    gt[2 * kChunk + 2 * lane + 1] = beta[2 * lane + 1];
    if (p.backward) {
      p.gsum[sh * kChunk + 2 * lane] = g0;
      p.gsum[sh * kChunk + 2 * lane + 1] = g1;
    }
  }
  __syncthreads();
  if (h % p.group == 0) {   // one of the heads that share these q, k stores their tiles
    const size_t at = ((size_t)c * p.hk + hk) * kQK;
    for (int i = tid * 16; i < kQK; i += 128 * 16) {
      *reinterpret_cast<uint4*>(p.kt + at + i) = *reinterpret_cast<const uint4*>(kt + i);
      *reinterpret_cast<uint4*>(p.qt + at + i) = *reinterpret_cast<const uint4*>(qt + i);
    }
  }
  float am[8][4], ap[8][4];
  zero(am);
  zero(ap);
  mma_tile<8, false, false, P, P, PS>(am, kt, kChunk, DKP, 16 * warp, kt, kChunk, DKP, 0, 0, DKP);
  mma_tile<8, false, false, P, P, PS>(ap, qt, kChunk, DKP, 16 * warp, kt, kChunk, DKP, 0, 0, DKP);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = 16 * warp + (lane >> 2) + 8 * r, cl = 8 * j + 2 * (lane & 3);
      const float d0 = cl <= i ? expf((float)(G[i] - G[cl])) : 0.f;
      const float d1 = cl + 1 <= i ? expf((float)(G[i] - G[cl + 1])) : 0.f;
      M[i * kMStride + cl] = cl < i ? am[j][2 * r] * d0 : 0.f;
      M[i * kMStride + cl + 1] = cl + 1 < i ? am[j][2 * r + 1] * d1 : 0.f;
      put2<PS>(pt, kChunk, kChunk, i, cl, cl <= i ? p.scale * ap[j][2 * r] * d0 : 0.f,
               cl + 1 <= i ? p.scale * ap[j][2 * r + 1] * d1 : 0.f);
    }
  __syncthreads();
  if (tid < kChunk) {
    float y[kChunk];   // beta_l X_lj
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      float s0 = M[i * kMStride + tid], s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
      for (int l = 0; l < (i & ~3); l += 4) {
        const float4 m = *reinterpret_cast<const float4*>(M + i * kMStride + l);
        s0 += m.x * y[l];
        s1 += m.y * y[l + 1];
        s2 += m.z * y[l + 2];
        s3 += m.w * y[l + 3];
      }
#pragma unroll
      for (int l = i & ~3; l < i; ++l) s1 += M[i * kMStride + l] * y[l];
      float x = -((s0 + s1) + (s2 + s3));
      y[i] = beta[i] * x;
#pragma unroll
      for (int q = 0; q < PS; ++q) {
        const __nv_bfloat16 hx = __float2bfloat16_rn(x);
        *reinterpret_cast<__nv_bfloat16*>(xt + tile_off(kChunk, i, q * kChunk + tid)) = hx;
        x -= __bfloat162float(hx);
        if (q == 0 && !(fabsf(x) <= 3.4e38f)) x = 0.f;
      }
    }
  } else {
    for (int i = (tid - kChunk) * 16; i < kXP; i += kChunk * 16)
      *reinterpret_cast<uint4*>(p.pt + sh * kXP + i) = *reinterpret_cast<const uint4*>(pt + i);
  }
  __syncthreads();
  for (int i = tid * 16; i < kXP; i += 128 * 16)
    *reinterpret_cast<uint4*>(p.xt + sh * kXP + i) = *reinterpret_cast<const uint4*>(xt + i);
}

template <int DKP, typename T, int PS>
cudaError_t run_prep(const Params& p, cudaStream_t s) {
  const auto fits = [&](const void* x, const Strides& st) {
    const int64_t v = 16 / (int64_t)sizeof(T);
    return (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && st.b % v == 0 && st.t % v == 0 && st.h % v == 0;
  };
  const bool dk_ok = p.dk % (16 / (int)sizeof(T)) == 0;
  const int vec = (dk_ok && fits(p.k, p.ks) ? 1 : 0) | (dk_ok && fits(p.q, p.qs) ? 2 : 0) | (fits(p.v, p.vs) ? 4 : 0) |
                  (fits(p.d_o, p.dos) ? 8 : 0);
  constexpr int smem = prep_smem<DKP, T, PS>();
  cudaError_t e = allow_smem(prep_kernel<DKP, T, PS>, smem);
  if (e != cudaSuccess) return e;
  const double tokens = (double)p.bound * kChunk;
  LaunchTimer t("delta_prep_kernel", s, tokens * p.hv * (2.0 * p.dk * sizeof(T) + 4.0 * kChunk * PS),
                tokens * p.hv * 4.0 * kChunk * p.dk);
  prep_kernel<DKP, T, PS><<<dim3((unsigned)p.bound, (unsigned)p.hv), 128, smem, s>>>(p, vec);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_plan(const Params& p, cudaStream_t s) {
  LaunchTimer t("delta_plan_kernel", s, 4.0 * p.nseq, 0);
  plan_kernel<<<1, 1024, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int PS>
static cudaError_t pick_prep(const Params& p, cudaStream_t s) {
  return p.dk <= 64 ? run_prep<64, T, PS>(p, s) : run_prep<128, T, PS>(p, s);
}

cudaError_t launch_prep(const Params& p, int dtype, cudaStream_t s) {
  constexpr int B = kBackPieces;
  if (dtype == 1) return p.backward ? pick_prep<__nv_bfloat16, B>(p, s) : pick_prep<__nv_bfloat16, 2>(p, s);
  if (dtype == 2) return p.backward ? pick_prep<__half, B>(p, s) : pick_prep<__half, 2>(p, s);
  return pick_prep<float, 3>(p, s);
}

}  // namespace delta
}  // namespace qrb
