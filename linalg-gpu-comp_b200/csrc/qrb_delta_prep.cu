// Per-chunk factors of the gated delta rule (mathematics in qrb_delta.cuh).
//
//   plan_kernel  packed layout: first chunk slot of every sequence (one block, a prefix sum).
//   prep_kernel  one block per (chunk, value head): the running decays, X and P of the chunk, and
//                the chunk's q, k, v (and dO) as zero-padded tiles.  These depend on no state, so all
//                chunks run at once and the sequential kernels are left with products only.
//
// X is a triangular inverse, as T factors are: the four diagonal 16 x 16 blocks by substitution, a
// column a thread, then two merges X_10 = R + X_11 beta R with R = -(M_10 + M_10 beta X_00), all in
// fp32.  One substitution over 64 rows (2016 multiply-adds in a row on 64 threads) and an exponential
// for every entry of M and P took 370 us for 8896 chunks and heads of 128; the merges are a third of
// that chain, and off the diagonal blocks a decay is a product of two tabled factors.
// Measured: 347 us for 24 packed sequences of 16384 tokens with 32 heads of 128 x 128 in bf16, 1.0 GB; shared
// memory is 71% busy and half the issue slots are used.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

// to[s] = sum of count(0 .. s - 1), never above `most`; to[nseq] the whole sum.  One block of 1024.
template <typename F>
__device__ void prefix(int nseq, int64_t most, int32_t* to, int* part, F count) {
  const int tid = threadIdx.x, per = (nseq + 1023) / 1024;
  int64_t sum = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < nseq) sum += count(tid * per + i);
  part[tid] = (int)min(sum, most);
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    int64_t v = part[tid];
    if (tid >= o) v += part[tid - o];
    __syncthreads();
    part[tid] = (int)min(v, most);
    __syncthreads();
  }
  int64_t at = tid == 0 ? 0 : part[tid - 1];
  for (int i = 0; i < per; ++i) {
    const int s = tid * per + i;
    if (s >= nseq) break;
    to[s] = (int)at;
    at = min(at + count(s), most);
    if (s == nseq - 1) to[nseq] = (int)at;
  }
  __syncthreads();
}

__global__ void __launch_bounds__(1024) plan_kernel(Params p) {
  __shared__ int part[1024];
  const int tid = threadIdx.x;
  auto chunks = [&](int s) {
    int64_t b, t0, n;
    seq_range(p, s, b, t0, n);
    return (n + kChunk - 1) / kChunk;
  };
  prefix(p.nseq, p.bound, p.cstart, part, chunks);
  if (p.seg > 0) {
    // of the chunks that have a slot, in case wrong offsets gave more
    prefix(p.nseq, p.nsegs, p.segstart, part, [&](int s) {
      return (int64_t)max(1, (p.cstart[s + 1] - p.cstart[s] + p.seg - 1) / p.seg);
    });
    return;
  }
  // Longest first, so that no long sequence is left to run alone at the end (24 packed prompts on 148
  // SMs: 58 chunks on the busiest instead of 82); calls of more sequences than threads level out anyway.
  if (p.nseq > 1024) {
    for (int s = tid; s < p.nseq; s += 1024) p.order[s] = s;
    return;
  }
  int mine = 0;
  if (tid < p.nseq) mine = part[tid] = (int)chunks(tid);
  __syncthreads();
  if (tid < p.nseq) {
    int rank = 0;
    for (int s = 0; s < p.nseq; ++s) rank += part[s] > mine || (part[s] == mine && s < tid);
    p.order[rank] = tid;
  }
}

constexpr int kPrepThreads = 256;
constexpr int kMStride = 68;   // floats per row of M and X: rows stay 16-byte aligned, columns on distinct banks
constexpr int kRStride = 36;

template <int DKP, typename T, int PS, int PO>
struct PrepLayout {
  static constexpr int P = Pieces<T>::kIn;
  static constexpr int kQK = tile_bytes(kChunk, P, DKP), kXP = tile_bytes(kChunk, PS, kChunk), kPP = tile_bytes(kChunk, PO, kChunk);
  static_assert(PO <= PS, "overlay");
  // once the products are taken, over k and q: X's two 32 x 32 diagonal blocks (fp32), the right sides
  // of a merge, and the pieces of P, later those of X.  60 KB with bf16 operands: three blocks an SM.
  static constexpr int kOffS = 0, kOffR = 2 * 32 * kRStride * 4, kOffT = 16384;
  static_assert(kOffR + 32 * kRStride * 4 <= kOffT, "overlay");
  static constexpr int kOffM = 2 * kQK > kOffT + kXP ? 2 * kQK : kOffT + kXP;   // M, fp32
  static constexpr int kOffG = kOffM + kChunk * kMStride * 4;                   // G (fp64), beta, decay tables
  static constexpr int kBytes = kOffG + kChunk * 8 + kChunk * 4 + kChunk * 4 + 4 * kChunk * 4;
  static_assert(kBytes <= 232448, "shared memory of one block");
};

// kChunk rows of W values, 16-byte units dealt out over the block: every load of a thread is issued
// before the first is used (a loop of load and store waits for memory once a turn).  Rows and columns
// that do not exist read existing ones and become zero.
template <typename T, int W>
struct Rows {
  static constexpr int V = 16 / sizeof(T), kUnits = kChunk * (W / V) / kPrepThreads;
  static_assert(kUnits * kPrepThreads * V == kChunk * W, "whole turns");
  uint4 r[kUnits];
  __device__ __forceinline__ static int row(int u) { return (threadIdx.x + u * kPrepThreads) / (W / V); }
  __device__ __forceinline__ static int col(int u) { return (threadIdx.x + u * kPrepThreads) % (W / V) * V; }
  __device__ __forceinline__ void load(const T* x, int64_t stride, int len, int d, bool vec) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int rr = row(u), c = col(u);
      const T* from = x + (int64_t)min(rr, len - 1) * stride;
      if (vec && d % V == 0) {
        r[u] = __ldg(reinterpret_cast<const uint4*>(from + (c < d ? c : 0)));
      } else {
        alignas(16) T e[V];
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = __ldg(from + min(c + i, d - 1));
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (c + i >= d) e[i] = from_f<T>(0.f);
        r[u] = *reinterpret_cast<uint4*>(e);
      }
      if (rr >= len || c >= d) r[u] = make_uint4(0, 0, 0, 0);
    }
  }
  // as pieces into an operand tile
  __device__ __forceinline__ void put(unsigned char* tile) const {
    constexpr int P = Pieces<T>::kIn;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int rr = row(u), c = col(u);
      if (P == 1) {
        *reinterpret_cast<uint4*>(tile + tile_off(kChunk, rr, c)) = r[u];
      } else {
        const T* e = reinterpret_cast<const T*>(&r[u]);
#pragma unroll
        for (int i = 0; i < V; i += 2) put2<P>(tile, kChunk, W, rr, c + i, to_f(e[i]), to_f(e[i + 1]));
      }
    }
  }
  // as they are, dense rows
  __device__ __forceinline__ void keep(unsigned char* to) const {
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      *reinterpret_cast<uint4*>(to + (size_t)(threadIdx.x + u * kPrepThreads) * 16) = r[u];
  }
};

template <typename T>
__device__ void zero_rows(const Params& p, int idx, int h, int hk) {
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
      if (h % p.group == 0) {
        T* dq = static_cast<T*>(p.dq) + (t * p.hk + hk) * p.dk;
        T* dk = static_cast<T*>(p.dk_) + (t * p.hk + hk) * p.dk;
        for (int c = threadIdx.x; c < p.dk; c += blockDim.x) dq[c] = dk[c] = from_f<T>(0.f);
      }
      if (threadIdx.x == 0) p.dg[t * p.hv + h] = p.dbeta[t * p.hv + h] = 0.f;
    }
  }
}

// R -= (M diag(beta)) X over l in [l0, l0 + N): two rows and four columns a thread.
template <int N>
__device__ __forceinline__ void block_product(float (&r)[2][4], const float* m0, const float* m1, const float* beta,
                                              const float* x, int stride) {
#pragma unroll 8
  for (int l = 0; l < N; ++l) {
    const float4 y = *reinterpret_cast<const float4*>(x + l * stride);
    const float b = beta[l], a0 = m0[l] * b, a1 = m1[l] * b;
    r[0][0] += a0 * y.x;
    r[0][1] += a0 * y.y;
    r[0][2] += a0 * y.z;
    r[0][3] += a0 * y.w;
    r[1][0] += a1 * y.x;
    r[1][1] += a1 * y.y;
    r[1][2] += a1 * y.z;
    r[1][3] += a1 * y.w;
  }
}

template <int DKP, typename T, int PS, int PO>
__global__ void __launch_bounds__(kPrepThreads, Pieces<T>::kIn == 1 ? 3 : 2) prep_kernel(Params p, int vec) {
  using L = PrepLayout<DKP, T, PS, PO>;
  constexpr int P = L::P;
  extern __shared__ __align__(128) unsigned char sm[];
  unsigned char *kt = sm, *qt = sm + L::kQK, *xp = sm + L::kOffT;
  float* M = reinterpret_cast<float*>(sm + L::kOffM);
  float* X = reinterpret_cast<float*>(sm + L::kOffS);
  float* R = reinterpret_cast<float*>(sm + L::kOffR);
  double* G = reinterpret_cast<double*>(sm + L::kOffG);
  float* beta = reinterpret_cast<float*>(G + kChunk);
  float* down = beta + kChunk;     // exp(G_i - G before i's block of 16)
  float* across = down + kChunk;   // [block][j]: exp(G before the block - G_j)
  const int c = blockIdx.x, h = blockIdx.y, hk = h / p.group, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Chunk ch = chunk_at(p, c);
  if (ch.seq < 0) {
    if (p.zero_tail) zero_rows<T>(p, ch.idx, h, hk);
    return;
  }
  const size_t sh = slot_head(p, c, h);
  float g[2] = {0.f, 0.f}, bt[2] = {0.f, 0.f};
  if (warp == 0) {
    const int64_t gbase = ch.b * p.gs.b + ch.t0 * p.gs.t + h * p.gs.h;
    const int64_t bbase = ch.b * p.bs.b + ch.t0 * p.bs.t + h * p.bs.h;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = min(2 * lane + e, ch.len - 1);
      g[e] = __ldg(p.g + gbase + i * p.gs.t);
      bt[e] = __ldg(p.beta + bbase + i * p.bs.t);
    }
  }
  {
    Rows<T, DKP> k, q;
    k.load(static_cast<const T*>(p.k) + ch.b * p.ks.b + ch.t0 * p.ks.t + hk * p.ks.h, p.ks.t, ch.len, p.dk, vec & 1);
    q.load(static_cast<const T*>(p.q) + ch.b * p.qs.b + ch.t0 * p.qs.t + hk * p.qs.h, p.qs.t, ch.len, p.dk, vec & 2);
    k.put(kt);
    q.put(qt);
  }
  if (warp == 0) {
    // Running sums of g in fp64: differences of far apart sums keep their low bits.
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (2 * lane + e >= ch.len) g[e] = bt[e] = 0.f;
      if (g[e] < kMinLog) g[e] = kMinLog;
    }
    double s = (double)g[0] + (double)g[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const double last = __shfl_sync(0xffffffffu, s, 31);
    const double g1 = s, g0 = s - (double)g[1];
    // G before this lane's block of 16 (8 lanes)
    double before = __shfl_sync(0xffffffffu, s, (lane & ~7) == 0 ? 0 : (lane & ~7) - 1);
    if (lane < 8) before = 0.;
    G[2 * lane] = g0;
    G[2 * lane + 1] = g1;
    beta[2 * lane] = bt[0];
    beta[2 * lane + 1] = bt[1];
    down[2 * lane] = expf((float)(g0 - before));
    down[2 * lane + 1] = expf((float)(g1 - before));
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const double ref = __shfl_sync(0xffffffffu, s, 8 * i - 1);
      if (lane < 8 * i) {
        across[i * kChunk + 2 * lane] = expf((float)(ref - g0));
        across[i * kChunk + 2 * lane + 1] = expf((float)(ref - g1));
      }
    }
    float* gt = p.gates + sh * 3 * kChunk;
    gt[2 * lane] = expf((float)g0);
    gt[2 * lane + 1] = expf((float)g1);
    gt[kChunk + 2 * lane] = expf((float)(last - g0));
    gt[kChunk + 2 * lane + 1] = expf((float)(last - g1));
    gt[2 * kChunk + 2 * lane] = bt[0];
    gt[2 * kChunk + 2 * lane + 1] = bt[1];
    if (p.backward) {
      p.gsum[sh * kChunk + 2 * lane] = g0;
      p.gsum[sh * kChunk + 2 * lane + 1] = g1;
    }
  }
  __syncthreads();
  if (h % p.group == 0) {   // one of the heads that share these q, k stores their tiles
    const size_t at = ((size_t)c * p.hk + hk) * L::kQK;
    for (int i = tid * 16; i < L::kQK; i += kPrepThreads * 16) {
      *reinterpret_cast<uint4*>(p.kt + at + i) = *reinterpret_cast<const uint4*>(kt + i);
      *reinterpret_cast<uint4*>(p.qt + at + i) = *reinterpret_cast<const uint4*>(qt + i);
    }
  }
  {
    // warps 0-3: K K^T, warps 4-7: Q K^T, 16 rows each
    const int blk = warp & 3, m0 = 16 * blk;
    float acc[8][4];
    zero(acc);
    mma_tile<8, false, false, P, P, P == 1 ? 1 : 3>(acc, warp < 4 ? kt : qt, kChunk, DKP, m0, kt, kChunk, DKP, 0, 0, DKP);
    __syncthreads();   // k and q are read: their memory changes hands
    // decays: exact in the diagonal block, the product of two factors <= 1 (for g <= 0) before it
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = m0 + (lane >> 2) + 8 * r, cl = 8 * j + 2 * (lane & 3);
        float d0 = 0.f, d1 = 0.f;
        if (j < 2 * blk) {
          const float a = down[i];
          const float2 x = *reinterpret_cast<const float2*>(across + blk * kChunk + cl);
          d0 = a * x.x;
          d1 = a * x.y;
        } else if (j < 2 * blk + 2) {
          if (cl <= i) d0 = expf((float)(G[i] - G[cl]));
          if (cl + 1 <= i) d1 = expf((float)(G[i] - G[cl + 1]));
        }
        if (warp < 4) {
          *reinterpret_cast<float2*>(M + i * kMStride + cl) =
              make_float2(cl < i ? acc[j][2 * r] * d0 : 0.f, cl + 1 < i ? acc[j][2 * r + 1] * d1 : 0.f);
        } else {
          put2<PO>(xp, kChunk, kChunk, i, cl, cl <= i ? p.scale * acc[j][2 * r] * d0 : 0.f,
                   cl + 1 <= i ? p.scale * acc[j][2 * r + 1] * d1 : 0.f);
        }
      }
    }
  }
  __syncthreads();
  if (tid < kChunk) {
    // the four diagonal 16 x 16 blocks of X, a column a thread
    const int o = tid & ~15, j = tid & 15;
    float* to = X + (o >> 5) * 32 * kRStride + (o & 16) * (kRStride + 1);
    float y[16];   // beta x
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float* m = M + (o + i) * kMStride + o;
      float s0 = m[j], s1 = 0.f;
#pragma unroll
      for (int l = 0; l < i; ++l) {
        if (l & 1) s1 += m[l] * y[l];
        else s0 += m[l] * y[l];
      }
      const float x = -(s0 + s1);
      y[i] = beta[o + i] * x;
      to[i * kRStride + j] = x;
    }
  } else {
    for (int i = (tid - kChunk) * 16; i < L::kPP; i += (kPrepThreads - kChunk) * 16)
      *reinterpret_cast<uint4*>(p.pt + sh * L::kPP + i) = *reinterpret_cast<const uint4*>(xp + i);
  }
  __syncthreads();
  // v and dO as kChunk x 128 tiles, one per 128 value columns: what the recurrences then read needs no
  // test of rows, columns or alignment.  Two warps merge meanwhile; the blocks of X above the diagonal
  // are zeroed here too.
  float r[2][4];
  const int half = tid >> 5 & 1, t16 = tid & 31;   // threads 0 .. 63: 8 x 4 tiles of 2 x 4
  const int i16 = (t16 >> 2) * 2, j16 = (t16 & 3) * 4;
  float* X32 = X + half * 32 * kRStride;
  // 16 -> 32: X_10 = R + X_11 beta R, R = -(M_10 + M_10 beta X_00), in both halves of the chunk
  if (tid < 64) {
    const float *ma = M + (32 * half + 16 + i16) * kMStride + 32 * half, *mb = ma + kMStride;
    const float4 a = *reinterpret_cast<const float4*>(ma + j16), b = *reinterpret_cast<const float4*>(mb + j16);
    r[0][0] = a.x, r[0][1] = a.y, r[0][2] = a.z, r[0][3] = a.w;
    r[1][0] = b.x, r[1][1] = b.y, r[1][2] = b.z, r[1][3] = b.w;
    block_product<16>(r, ma, mb, beta + 32 * half, X32 + j16, kRStride);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float4*>(R + (16 * half + i16 + e) * kRStride + j16) =
          make_float4(-r[e][0], -r[e][1], -r[e][2], -r[e][3]);
    __syncwarp();   // each half is one warp's
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int q = 0; q < 4; ++q) r[e][q] = -r[e][q];
    const float* xa = X32 + (16 + i16) * kRStride + 16;
    block_product<16>(r, xa, xa + kRStride, beta + 32 * half + 16, R + 16 * half * kRStride + j16, kRStride);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float4*>(X32 + (16 + i16 + e) * kRStride + j16) =
          make_float4(r[e][0], r[e][1], r[e][2], r[e][3]);
  } else {
    for (int i = (tid - 64) * 16; i < L::kXP; i += (kPrepThreads - 64) * 16)
      *reinterpret_cast<uint4*>(xp + i) = make_uint4(0, 0, 0, 0);
  }
  for (int vb = 0; vb * 128 < p.dv; ++vb) {
    const size_t vat = (sh * ((p.dv + 127) / 128) + vb) * kChunk * 128 * sizeof(T);
    Rows<T, 128> v;
    v.load(static_cast<const T*>(p.v) + ch.b * p.vs.b + ch.t0 * p.vs.t + h * p.vs.h + vb * 128, p.vs.t, ch.len,
           min(128, p.dv - vb * 128), vec & 4);
    v.keep(p.vt + vat);
    if (p.backward) {
      v.load(static_cast<const T*>(p.d_o) + ch.b * p.dos.b + ch.t0 * p.dos.t + h * p.dos.h + vb * 128, p.dos.t, ch.len,
             min(128, p.dv - vb * 128), vec & 8);
      v.keep(p.dot + vat);
    }
  }
  __syncthreads();
  // 32 -> 64 the same way: 16 x 8 tiles of 2 x 4, the first 128 threads
  const int i32 = ((tid & 127) >> 3) * 2, j32 = (tid & 7) * 4;
  if (tid < 128) {
    const float *ma = M + (32 + i32) * kMStride, *mb = ma + kMStride;
    const float4 a = *reinterpret_cast<const float4*>(ma + j32), b = *reinterpret_cast<const float4*>(mb + j32);
    r[0][0] = a.x, r[0][1] = a.y, r[0][2] = a.z, r[0][3] = a.w;
    r[1][0] = b.x, r[1][1] = b.y, r[1][2] = b.z, r[1][3] = b.w;
    // X_00's columns 16 .. 31 begin at row 16
    if (j32 < 16)
      block_product<32>(r, ma, mb, beta, X + j32, kRStride);
    else
      block_product<16>(r, ma + 16, mb + 16, beta + 16, X + 16 * kRStride + j32, kRStride);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float4*>(R + (i32 + e) * kRStride + j32) = make_float4(-r[e][0], -r[e][1], -r[e][2], -r[e][3]);
  } else {
    // meanwhile: pieces of the two diagonal 32 x 32 blocks
    for (int u = tid - 128; u < 2 * 32 * 16; u += 128) {
      const int o = u >> 9, i = (u >> 4) & 31, j = (u & 15) * 2;
      if (j < i) {
        const float* x = X + (o * 32 + i) * kRStride + j;
        put2<PS>(xp, kChunk, kChunk, 32 * o + i, 32 * o + j, x[0], j + 1 < i ? x[1] : 0.f);
      }
    }
  }
  __syncthreads();
  if (tid < 128) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int q = 0; q < 4; ++q) r[e][q] = -r[e][q];
    const float* xa = X + (32 + i32) * kRStride;
    // X_11's rows 0 .. 15 have nothing in its second half's columns
    if (i32 < 16)
      block_product<16>(r, xa, xa + kRStride, beta + 32, R + j32, kRStride);
    else
      block_product<32>(r, xa, xa + kRStride, beta + 32, R + j32, kRStride);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      put2<PS>(xp, kChunk, kChunk, 32 + i32 + e, j32, r[e][0], r[e][1]);
      put2<PS>(xp, kChunk, kChunk, 32 + i32 + e, j32 + 2, r[e][2], r[e][3]);
    }
  }
  __syncthreads();
  for (int i = tid * 16; i < L::kXP; i += kPrepThreads * 16)
    *reinterpret_cast<uint4*>(p.xt + sh * L::kXP + i) = *reinterpret_cast<const uint4*>(xp + i);
}

template <int DKP, typename T, int PS, int PO>
cudaError_t run_prep(const Params& p, cudaStream_t s) {
  const auto fits = [&](const void* x, const Strides& st) {
    const int64_t v = 16 / (int64_t)sizeof(T);
    return (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && st.b % v == 0 && st.t % v == 0 && st.h % v == 0;
  };
  const bool dk_ok = p.dk % (16 / (int)sizeof(T)) == 0;
  const int vec = (dk_ok && fits(p.k, p.ks) ? 1 : 0) | (dk_ok && fits(p.q, p.qs) ? 2 : 0) | (fits(p.v, p.vs) ? 4 : 0) |
                  (fits(p.d_o, p.dos) ? 8 : 0);
  constexpr int smem = PrepLayout<DKP, T, PS, PO>::kBytes;
  cudaError_t e = allow_smem<prep_kernel<DKP, T, PS, PO>>(smem);
  if (e != cudaSuccess) return e;
  const double tokens = (double)p.bound * kChunk;
  LaunchTimer t("delta_prep_kernel", s, tokens * (2.0 * p.hk * p.dk * sizeof(T) + p.hv * (2.0 * kChunk * (PS + PO) + p.dv * sizeof(T))),
                tokens * p.hv * 4.0 * kChunk * p.dk);
  prep_kernel<DKP, T, PS, PO><<<dim3((unsigned)p.bound, (unsigned)p.hv), kPrepThreads, smem, s>>>(p, vec);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_plan(const Params& p, cudaStream_t s) {
  LaunchTimer t("delta_plan_kernel", s, 4.0 * p.nseq, 0);
  plan_kernel<<<1, 1024, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int PS, int PO>
static cudaError_t pick_prep(const Params& p, cudaStream_t s) {
  return p.dk <= 64 ? run_prep<64, T, PS, PO>(p, s) : run_prep<128, T, PS, PO>(p, s);
}

cudaError_t launch_prep(const Params& p, int dtype, cudaStream_t s) {
  constexpr int B = kBackPieces;
  constexpr int C = kChainPieces;
  if (dtype == 1) return p.backward ? pick_prep<__nv_bfloat16, C, B>(p, s) : pick_prep<__nv_bfloat16, C, 2>(p, s);
  if (dtype == 2) return p.backward ? pick_prep<__half, C, B>(p, s) : pick_prep<__half, C, 2>(p, s);
  return pick_prep<float, 3, 3>(p, s);
}

}  // namespace delta
}  // namespace qrb
