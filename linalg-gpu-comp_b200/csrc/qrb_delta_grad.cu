// Gradients of q, k, g and beta of the gated delta rule, chunk by chunk (mathematics in
// qrb_delta.cuh), with mma.sync: for fp32, whose three pieces leave no room for tiles in flight beside
// tcgen05's operands.  qrb_delta_gradtc.cu has the 16-bit types.
//
// With every chunk's S0, e, dS' and du in the workspace the chunks are independent: one block
// per (chunk, q/k head) adds the heads that share it in order, so no atomics are needed and
// results repeat.  Value columns pass through in tiles of 32 by cp.async, one at a time; 16 warps hold, as
// 16 x 32 pieces, the products with S0 and dS' (kept apart: their rows scale differently) and
// 16 x 16 pieces of dO e^T and du e^T, which then meet K and Q.  beta is applied to rows and
// columns of products, so that e and du serve as they are.  The sums dg and dbeta are made of come
// from the recurrences; here they are added up in order.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

template <int DKP>
struct GLayout {
  static constexpr int P = kBackPieces;                     // of the inputs as of what the recurrences leave
  static_assert(P == Pieces<float>::kIn && P == Pieces<float>::kS, "three pieces throughout");
  static constexpr int kK = tile_bytes(kChunk, P, DKP);
  static constexpr int kS = tile_bytes(kTile, P, DKP);      // S0, dS': value columns as rows
  static constexpr int kF = tile_bytes(kTile, P, kChunk);   // e, du: the same
  static constexpr int kD = tile_bytes(kChunk, P, kTile);
  static constexpr int kOffE = 0, kOffDU = kF, kOffS0 = 2 * kF, kOffDS = kOffS0 + kS, kOffD = kOffDS + kS;
  static constexpr int kTile32 = kOffD + kD;                // the operands of 32 value columns
  static constexpr int kZ = tile_bytes(kChunk, P, kChunk);
  static constexpr int kOffQ = kK, kOffT = 2 * kK;
  // Z and N are formed when the last tile is consumed and lie over it
  static constexpr int kTiles = kTile32 > 2 * kZ ? kTile32 : 2 * kZ;
  static constexpr int kOffG = kOffT + kTiles;     // G (64 doubles), gates, row sums, reductions
  static constexpr int kBytes = kOffG + 64 * 8 + 3 * 64 * 4;
};

template <int DKP>
__global__ void __launch_bounds__(512) grad_kernel(Params p) {
  using L = GLayout<DKP>;
  constexpr int P = L::P;
  constexpr int NT = DKP / 32;           // 8-column blocks of q / k columns a warp holds
  extern __shared__ __align__(128) unsigned char sm[];
  unsigned char *K = sm, *Q = sm + L::kOffQ, *TT = sm + L::kOffT;
  unsigned char *Z = TT, *N = TT + L::kZ;
  double* G = reinterpret_cast<double*>(sm + L::kOffG);
  float* gates = reinterpret_cast<float*>(G + 64);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int c = blockIdx.x, hk = blockIdx.y;
  const int m0 = 16 * (warp & 3), cq = warp >> 2, d0 = cq * (DKP / 4);
  const Chunk ch = chunk_at(p, c);
  if (ch.seq < 0) return;
  {
    const size_t at = ((size_t)c * p.hk + hk) * L::kK;
    cp_tile(K, p.kt + at, L::kK);
    cp_tile(Q, p.qt + at, L::kK);
    cp_commit();
  }
  float tq_[NT][4], tk_[NT][4];          // sums over the heads of the group
  zero(tq_);
  zero(tk_);
  for (int hh = 0; hh < p.group; ++hh) {
    const int h = hk * p.group + hh;
    const size_t at = slot_head(p, c, h);
    auto dO = [&](int n) {   // the tile's columns of dO, kLanes values a token
      return reinterpret_cast<const float*>(p.dot) + (at * ((p.dv + kLanes - 1) / kLanes) + n / 4) * kChunk * kLanes + n % 4 * kTile;
    };
    __syncthreads();                     // the previous head's Z, N and sums are consumed
    if (tid < 64) G[tid] = p.gsum[at * 64 + tid];
    if (tid < 192) gates[tid] = p.gates[at * 192 + tid];
    float aq[NT][4], ay[NT][4], au[NT][4], az[2][4], an[2][4];
    zero(aq);
    zero(ay);
    zero(au);
    zero(az);
    zero(an);
    unsigned char *E = TT + L::kOffE, *DU = TT + L::kOffDU, *S0 = TT + L::kOffS0, *DS = TT + L::kOffDS, *D = TT + L::kOffD;
    for (int n = 0; n < p.nv; ++n) {
      float x[4];
      const float* from = dO(n) + (size_t)(tid >> 3) * kLanes + (tid & 7) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __ldg(from + i);
      __syncthreads();                   // the previous tile is consumed
      const size_t t = at * p.nv + n;
      cp_tile(E, p.ep + t * L::kF, L::kF);
      cp_tile(DU, p.dup + t * L::kF, L::kF);
      cp_tile(S0, p.s0p + t * L::kS, L::kS);
      cp_tile(DS, p.dsp + t * L::kS, L::kS);
      cp_commit();
      cp_wait_all();
      put2<P>(D, kChunk, kTile, tid >> 3, (tid & 7) * 4, x[0], x[1]);
      put2<P>(D, kChunk, kTile, tid >> 3, (tid & 7) * 4 + 2, x[2], x[3]);
      __syncthreads();
      mma_tile<NT, false, true, P, P, P, false, true>(aq, D, kChunk, kTile, m0, S0, kTile, DKP, d0, 0, kTile);
      mma_tile<NT, true, true, P, P, P, true, true>(ay, DU, kTile, kChunk, m0, S0, kTile, DKP, d0, 0, kTile);
      mma_tile<NT, true, true, P, P, P, true, true>(au, E, kTile, kChunk, m0, DS, kTile, DKP, d0, 0, kTile);
      if (16 * cq <= m0) {               // Z, N are lower triangular
        mma_tile<2, false, true, P, P, P, false, true>(az, D, kChunk, kTile, m0, E, kTile, kChunk, 16 * cq, 0, kTile);
        mma_tile<2, true, true, P, P, P, true, true>(an, DU, kTile, kChunk, m0, E, kTile, kChunk, 16 * cq, 0, kTile);
      }
    }
    __syncthreads();                     // tiles consumed: Z and N may overwrite them
    const float* gam = gates;
    const float* tail = gates + 64;
    const float* bet = gates + 128;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = m0 + gr + 8 * r, l = 16 * cq + 8 * j + 2 * tq;
        float z[2], w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float dc = l + e <= i ? expf((float)(G[i] - G[l + e])) * bet[l + e] : 0.f;
          z[e] = l + e <= i ? p.scale * dc * az[j][2 * r + e] : 0.f;
          w[e] = l + e < i ? -dc * bet[i] * an[j][2 * r + e] : 0.f;
        }
        put2<P>(Z, kChunk, kChunk, i, l, z[0], z[1]);
        put2<P>(N, kChunk, kChunk, i, l, w[0], w[1]);
      }
    // row scalings
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = m0 + gr + 8 * (r >> 1);
        aq[j][r] *= p.scale * gam[i];
        ay[j][r] = tail[i] * bet[i] * au[j][r] - gam[i] * bet[i] * ay[j][r];
      }
    __syncthreads();
    mma_tile<NT, false, true, P, P, P>(aq, Z, kChunk, kChunk, m0, K, kChunk, DKP, d0, 0, m0 + 16);
    mma_tile<NT, true, true, P, P, P>(ay, Z, kChunk, kChunk, m0, Q, kChunk, DKP, d0, m0, kChunk);
    mma_tile<NT, false, true, P, P, P>(ay, N, kChunk, kChunk, m0, K, kChunk, DKP, d0, 0, m0 + 16);
    mma_tile<NT, true, true, P, P, P>(ay, N, kChunk, kChunk, m0, K, kChunk, DKP, d0, m0, kChunk);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        tq_[j][r] += aq[j][r];
        tk_[j][r] += ay[j][r];
      }
    if (warp == 0) gate_sums(p, ch, at, h, lane);
  }
  const int64_t tok = ch.b * p.time + ch.t0;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = m0 + gr + 8 * (r >> 1), col = d0 + 8 * j + 2 * tq + (r & 1);
      if (i < ch.len && col < p.dk) {
        const size_t at = ((size_t)(tok + i) * p.hk + hk) * p.dk + col;
        static_cast<float*>(p.dq)[at] = tq_[j][r];
        static_cast<float*>(p.dk_)[at] = tk_[j][r];
      }
    }
}

template <int DKP>
cudaError_t run_grad(const Params& p, cudaStream_t s) {
  constexpr int smem = GLayout<DKP>::kBytes;
  static_assert(smem <= 232448, "shared memory of one block");
  const double rows = (double)p.bound * kChunk * p.hv;
  LaunchTimer t("delta_grad_kernel", s, rows * 4.0 * p.dk * sizeof(float), rows * (6.0 * p.dv + 8.0 * kChunk) * p.dk);
  cudaError_t e = allow_smem<grad_kernel<DKP>>(smem);
  if (e != cudaSuccess) return e;
  grad_kernel<DKP><<<dim3((unsigned)p.bound, (unsigned)p.hk), 512, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_grad(const Params& p, int dtype, cudaStream_t s) {
  if (grad_on_tc(dtype)) return dtype == 1 ? launch_grad_tc<__nv_bfloat16>(p, s) : launch_grad_tc<__half>(p, s);
  return p.dk <= 64 ? run_grad<64>(p, s) : run_grad<128>(p, s);
}

}  // namespace delta
}  // namespace qrb
