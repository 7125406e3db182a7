// Gradients of q, k, g and beta of the gated delta rule, chunk by chunk (mathematics in
// qrb_delta.cuh), with mma.sync: for fp32, whose three pieces leave no room for tiles in flight beside
// tcgen05's operands.  qrb_delta_gradtc.cu has the 16-bit types.
//
// With every chunk's S0, e, dS' and du in the workspace the chunks are independent: one block
// per (chunk, q/k head) adds the heads that share it in order, so no atomics are needed and
// results repeat.  Value columns pass through in tiles of 32 by cp.async; 16 warps hold, as
// 16 x 32 pieces, the products with S0 and dS' (kept apart: their rows scale differently) and
// 16 x 16 pieces of dO e^T and du e^T, which then meet K and Q.  beta is applied to rows and
// columns of products, so that e and du serve as they are.  The sums dg and dbeta are made of come
// from the recurrences; here they are added up in order.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

template <int DKP, typename T>
struct GLayout {
  static constexpr int P = Pieces<T>::kIn, PS = Pieces<T>::kS;
  static constexpr int kStages = PS == 2 ? 2 : 1;
  static constexpr int kK = tile_bytes(kChunk, P, DKP);
  static constexpr int kS = tile_bytes(kTile, PS, DKP);      // S0, dS': value columns as rows
  static constexpr int kF = tile_bytes(kTile, PS, kChunk);   // e, du: the same
  static constexpr int kD = tile_bytes(kChunk, P, kTile);
  // tiles in the workspace have kBackPieces pieces; the first kS of them are a prefix
  static constexpr int kWS = tile_bytes(kTile, kBackPieces, DKP), kWF = tile_bytes(kTile, kBackPieces, kChunk);
  static constexpr int kOffE = 0, kOffDU = kF, kOffS0 = 2 * kF, kOffDS = kOffS0 + kS, kOffD = kOffDS + kS;
  static constexpr int kStage = kOffD + kD;
  static constexpr int kZ = tile_bytes(kChunk, PS, kChunk);
  static constexpr int kOffQ = kK, kOffT = 2 * kK;
  // Z and N are formed when the last tile is consumed and lie over the tiles
  static constexpr int kTiles = kStages * kStage > 2 * kZ ? kStages * kStage : 2 * kZ;
  static constexpr int kOffG = kOffT + kTiles;     // G (64 doubles), gates, row sums, reductions
  static constexpr int kBytes = kOffG + 64 * 8 + 3 * 64 * 4;
};

template <int DKP, typename T>
__global__ void __launch_bounds__(512) grad_kernel(Params p) {
  using L = GLayout<DKP, T>;
  constexpr int P = L::P, PS = L::PS;
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
      return reinterpret_cast<const T*>(p.dot) + (at * ((p.dv + kLanes - 1) / kLanes) + n / 4) * kChunk * kLanes + n % 4 * kTile;
    };
    auto load = [&](int n, int stage) {
      unsigned char* d = TT + stage * L::kStage;
      const size_t t = at * p.nv + n;
      cp_tile(d + L::kOffE, p.ep + t * L::kWF, L::kF);
      cp_tile(d + L::kOffDU, p.dup + t * L::kWF, L::kF);
      cp_tile(d + L::kOffS0, p.s0p + t * L::kWS, L::kS);
      cp_tile(d + L::kOffDS, p.dsp + t * L::kWS, L::kS);
      // dO: 32 columns of the staged tile, which bf16 tiles take unit by unit
      if (P == 1 && tid < 4 * kChunk)
        cp16(d + L::kOffD + tile_off(kChunk, tid >> 2, (tid & 3) * 8), dO(n) + (size_t)(tid >> 2) * kLanes + (tid & 3) * 8);
      cp_commit();
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
    if (L::kStages == 2) load(0, 0);
    for (int n = 0; n < p.nv; ++n) {
      const int stage = L::kStages == 2 ? (n & 1) : 0;
      unsigned char* d = TT + stage * L::kStage;
      const unsigned char *E = d + L::kOffE, *DU = d + L::kOffDU, *S0 = d + L::kOffS0, *DS = d + L::kOffDS;
      unsigned char* D = d + L::kOffD;
      T x[4];
      if (P > 1) {
        const T* from = dO(n) + (size_t)(tid >> 3) * kLanes + (tid & 7) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __ldg(from + i);
      }
      if (L::kStages == 2) {
        cp_wait_all();
        __syncthreads();
        if (n + 1 < p.nv) load(n + 1, stage ^ 1);
      } else {
        __syncthreads();
        load(n, 0);
        cp_wait_all();
      }
      if (P > 1) {
        put2<P>(D, kChunk, kTile, tid >> 3, (tid & 7) * 4, to_f(x[0]), to_f(x[1]));
        put2<P>(D, kChunk, kTile, tid >> 3, (tid & 7) * 4 + 2, to_f(x[2]), to_f(x[3]));
      }
      if (P > 1 || L::kStages == 1) __syncthreads();
      mma_tile<NT, false, true, P, PS, PS, false, true>(aq, D, kChunk, kTile, m0, S0, kTile, DKP, d0, 0, kTile);
      mma_tile<NT, true, true, PS, PS, PS, true, true>(ay, DU, kTile, kChunk, m0, S0, kTile, DKP, d0, 0, kTile);
      mma_tile<NT, true, true, PS, PS, PS, true, true>(au, E, kTile, kChunk, m0, DS, kTile, DKP, d0, 0, kTile);
      if (16 * cq <= m0) {               // Z, N are lower triangular
        mma_tile<2, false, true, P, PS, PS, false, true>(az, D, kChunk, kTile, m0, E, kTile, kChunk, 16 * cq, 0, kTile);
        mma_tile<2, true, true, PS, PS, PS, true, true>(an, DU, kTile, kChunk, m0, E, kTile, kChunk, 16 * cq, 0, kTile);
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
        put2<PS>(Z, kChunk, kChunk, i, l, z[0], z[1]);
        put2<PS>(N, kChunk, kChunk, i, l, w[0], w[1]);
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
    mma_tile<NT, false, true, PS, P, PS>(aq, Z, kChunk, kChunk, m0, K, kChunk, DKP, d0, 0, m0 + 16);
    mma_tile<NT, true, true, PS, P, PS>(ay, Z, kChunk, kChunk, m0, Q, kChunk, DKP, d0, m0, kChunk);
    mma_tile<NT, false, true, PS, P, PS>(ay, N, kChunk, kChunk, m0, K, kChunk, DKP, d0, 0, m0 + 16);
    mma_tile<NT, true, true, PS, P, PS>(ay, N, kChunk, kChunk, m0, K, kChunk, DKP, d0, m0, kChunk);
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
        static_cast<T*>(p.dq)[at] = from_f<T>(tq_[j][r]);
        static_cast<T*>(p.dk_)[at] = from_f<T>(tk_[j][r]);
      }
    }
}

template <int DKP, typename T>
cudaError_t run_grad(const Params& p, cudaStream_t s) {
  constexpr int smem = GLayout<DKP, T>::kBytes;
  static_assert(smem <= 232448, "shared memory of one block");
  const double rows = (double)p.bound * kChunk * p.hv;
  LaunchTimer t("delta_grad_kernel", s, rows * 4.0 * p.dk * sizeof(T), rows * (6.0 * p.dv + 8.0 * kChunk) * p.dk);
  cudaError_t e = allow_smem<grad_kernel<DKP, T>>(smem);
  if (e != cudaSuccess) return e;
  grad_kernel<DKP, T><<<dim3((unsigned)p.bound, (unsigned)p.hk), 512, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_grad(const Params& p, int dtype, cudaStream_t s) {
  if (grad_on_tc(dtype)) return dtype == 1 ? launch_grad_tc<__nv_bfloat16>(p, s) : launch_grad_tc<__half>(p, s);
  return p.dk <= 64 ? run_grad<64, float>(p, s) : run_grad<128, float>(p, s);
}

}  // namespace delta
}  // namespace qrb
