// The forward recurrence of the gated delta rule over the chunks of one sequence
// (mathematics in qrb_delta.cuh).
//
// The columns of the state evolve independently, so a block owns one (sequence, value head,
// 32-column tile) and walks its chunks: the state tile stays in the accumulators of the last
// product for the whole sequence, and its pieces in shared memory.  Per chunk three dependent
// products, K S0, X F and K^T U, with two block barriers between them; the output's products
// Q S0 (sharing the fragments of S0) and P U fill the tensor pipe beside them.  The operand
// tiles of the next chunk arrive by cp.async meanwhile.  32 columns: a narrower tile repeats
// the loads of K, Q, X, P more often, a wider one leaves too few blocks for a single sequence.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

template <int DKP, typename T, int PS>
struct ScanLayout {
  static constexpr int P = Pieces<T>::kIn;
  static constexpr int kK = tile_bytes(kChunk, P, DKP);
  static constexpr int kX = tile_bytes(kChunk, PS, kChunk);
  static constexpr int kGates = 3 * kChunk * 4;
  static constexpr int kOffQ = kK, kOffX = 2 * kK, kOffP = kOffX + kX, kOffG = kOffP + kX;
  static constexpr int kStage = kOffG + 1024;
  static constexpr int kS = tile_bytes(DKP, PS, kTile);
  static constexpr int kF = tile_bytes(kChunk, PS, kTile);
  // two stages where they fit: not with two- or three-piece q and k of 128 columns
  static constexpr int kStages = 2 * kStage + kS + 3 * kF <= 232448 ? 2 : 1;
  static constexpr int kOffS = kStages * kStage, kOffF = kOffS + kS, kOffU = kOffF + kF, kOffT = kOffU + kF;
  static constexpr int kBytes = kOffT + kF;
  static_assert(kBytes <= 232448, "shared memory of one block");
};

// STORE: for a backward pass, keep the chunk's first state, e and the sums o.do instead of o.
template <int DKP, typename T, int PS, bool STORE>
__global__ void __launch_bounds__(256) scan_kernel(Params p) {
  using L = ScanLayout<DKP, T, PS>;
  constexpr int P = L::P;
  constexpr int SNT = DKP == 128 ? 4 : 2;   // 8-column blocks of the state a warp holds
  extern __shared__ __align__(128) unsigned char sm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int tile = blockIdx.x % p.nv, sh = blockIdx.x / p.nv, h = sh % p.hv, seq = sh / p.hv;
  const int hk = h / p.group, n0 = tile * kTile;
  const int sm0 = DKP == 128 ? 16 * warp : 16 * (warp & 3), sn0 = DKP == 128 ? 0 : 16 * (warp >> 2);
  const int m0 = 16 * (warp & 3), c0 = 16 * (warp >> 2);   // token rows, value columns of the other products
  unsigned char *S = sm + L::kOffS, *F = sm + L::kOffF, *U = sm + L::kOffU, *W = sm + L::kOffT;
  int64_t b, t0, n;
  seq_range(p, seq, b, t0, n);
  int slot0, nc;
  seq_slots(p, seq, slot0, nc);

  float st[SNT][4];
  const size_t sbase = ((size_t)seq * p.hv + h) * p.dk * p.dv;
#pragma unroll
  for (int j = 0; j < SNT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = sm0 + gr + 8 * (r >> 1), col = n0 + sn0 + 8 * j + 2 * tq + (r & 1);
      st[j][r] = p.s_init != nullptr && row < p.dk && col < p.dv ? p.s_init[sbase + (size_t)row * p.dv + col] : 0.f;
    }
  auto put_state = [&] {
#pragma unroll
    for (int j = 0; j < SNT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        put2<PS>(S, DKP, kTile, sm0 + gr + 8 * r, sn0 + 8 * j + 2 * tq, st[j][2 * r], st[j][2 * r + 1]);
  };
  auto load = [&](int c, int stage) {
    unsigned char* d = sm + stage * L::kStage;
    const size_t qk = ((size_t)(slot0 + c) * p.hk + hk) * L::kK, at = slot_head(p, slot0 + c, h);
    cp_tile(d, p.kt + qk, L::kK);
    cp_tile(d + L::kOffQ, p.qt + qk, L::kK);
    cp_tile(d + L::kOffX, p.xt + at * L::kX, L::kX);
    cp_tile(d + L::kOffP, p.pt + at * L::kX, L::kX);
    cp_tile(d + L::kOffG, reinterpret_cast<const unsigned char*>(p.gates + at * 3 * kChunk), L::kGates);
    cp_commit();
  };
  put_state();
  if (L::kStages == 2 && nc > 0) load(0, 0);
  for (int c = 0; c < nc; ++c) {
    const int stage = L::kStages == 2 ? (c & 1) : 0;
    unsigned char* d = sm + stage * L::kStage;
    const float* gates = reinterpret_cast<const float*>(d + L::kOffG);
    const int64_t left = n - (int64_t)c * kChunk;
    const int len = left < kChunk ? (int)left : kChunk;
    const int64_t tok = t0 + (int64_t)c * kChunk;
    // this thread's values: rows m0 + gr (+ 8), columns c0 + 8 j + 2 tq (+ 1)
    float v[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = m0 + gr + 8 * (r >> 1), col = n0 + c0 + 8 * j + 2 * tq + (r & 1);
        v[j][r] = row < len && col < p.dv
                      ? to_f(static_cast<const T*>(p.v)[b * p.vs.b + (tok + row) * p.vs.t + h * p.vs.h + col])
                      : 0.f;
      }
    if (L::kStages == 2) {
      cp_wait_all();
      __syncthreads();   // this chunk's tiles and the state are in place, the other stage is free
      if (c + 1 < nc) load(c + 1, stage ^ 1);
    } else {
      __syncthreads();
      load(c, 0);
      cp_wait_all();
      __syncthreads();
    }
    if (STORE) {
      unsigned char* to = p.s0p + (slot_head(p, slot0 + c, h) * p.nv + tile) * L::kS;
      for (int i = tid * 16; i < L::kS; i += 256 * 16)
        *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(S + i);
    }
    float e[2][4], o[2][4];
    zero(e);
    mma_tile<2, false, true, P, PS, PS>(e, d, kChunk, DKP, m0, S, DKP, kTile, c0, 0, DKP);
    zero(o);
    mma_tile<2, false, true, P, PS, PS>(o, d + L::kOffQ, kChunk, DKP, m0, S, DKP, kTile, c0, 0, DKP);
    float gam[2], tail[2], bet[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = m0 + gr + 8 * r;
      gam[r] = gates[i];
      tail[r] = gates[kChunk + i];
      bet[r] = gates[2 * kChunk + i];
    }
    const float glast = gates[kChunk - 1];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        e[j][2 * r] = v[j][2 * r] - gam[r] * e[j][2 * r];
        e[j][2 * r + 1] = v[j][2 * r + 1] - gam[r] * e[j][2 * r + 1];
        put2<PS>(F, kChunk, kTile, m0 + gr + 8 * r, c0 + 8 * j + 2 * tq, bet[r] * e[j][2 * r],
                 bet[r] * e[j][2 * r + 1]);
      }
    __syncthreads();
    // X is lower triangular: nothing right of this warp's rows
    mma_tile<2, false, true, PS, PS, PS>(e, d + L::kOffX, kChunk, kChunk, m0, F, kChunk, kTile, c0, 0, m0 + 16);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = m0 + gr + 8 * r, col = c0 + 8 * j + 2 * tq;
        if (STORE)
          put2<PS>(p.ep + (slot_head(p, slot0 + c, h) * p.nv + tile) * L::kF, kChunk, kTile, row, col, e[j][2 * r],
                   e[j][2 * r + 1]);
        const float u0 = bet[r] * e[j][2 * r], u1 = bet[r] * e[j][2 * r + 1];
        put2<PS>(U, kChunk, kTile, row, col, u0, u1);
        put2<PS>(W, kChunk, kTile, row, col, tail[r] * u0, tail[r] * u1);
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SNT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[j][r] *= glast;
    mma_tile<SNT, true, true, P, PS, PS>(st, d, kChunk, DKP, sm0, W, kChunk, kTile, sn0, 0, kChunk);
    put_state();
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[j][r] *= p.scale * gam[r >> 1];
    mma_tile<2, false, true, PS, PS, PS>(o, d + L::kOffP, kChunk, kChunk, m0, U, kChunk, kTile, c0, 0, m0 + 16);
    float dot[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = m0 + gr + 8 * (r >> 1), col = n0 + c0 + 8 * j + 2 * tq + (r & 1);
        if (row < len && col < p.dv) {
          if (STORE)
            dot[r >> 1] += o[j][r] * to_f(static_cast<const T*>(p.d_o)[b * p.dos.b + (tok + row) * p.dos.t +
                                                                       h * p.dos.h + col]);
          else
            static_cast<T*>(p.o)[b * p.os.b + (tok + row) * p.os.t + h * p.os.h + col] = from_f<T>(o[j][r]);
        }
      }
    if (STORE) {   // the two column halves of a row belong to two warps
      float* sums = p.odo + ((slot_head(p, slot0 + c, h) * p.nv + tile) * 2 + (warp >> 2)) * kChunk;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], 1);
        dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], 2);
        if (tq == 0) sums[m0 + gr + 8 * r] = dot[r];
      }
    }
  }
  if (p.s_end != nullptr) {
#pragma unroll
    for (int j = 0; j < SNT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = sm0 + gr + 8 * (r >> 1), col = n0 + sn0 + 8 * j + 2 * tq + (r & 1);
        if (row < p.dk && col < p.dv) p.s_end[sbase + (size_t)row * p.dv + col] = st[j][r];
      }
  }
}

template <int DKP, typename T, int PS, bool STORE>
cudaError_t run_scan(const Params& p, cudaStream_t s) {
  constexpr int smem = ScanLayout<DKP, T, PS>::kBytes;
  const unsigned grid = (unsigned)p.nseq * p.hv * p.nv;
  const double rows = (double)p.bound * kChunk * p.hv;
  LaunchTimer t(STORE ? "delta_scan_store_kernel" : "delta_scan_kernel", s, rows * 2.0 * p.dv * sizeof(T),
                rows * 6.0 * p.dk * p.dv);
  cudaError_t e = allow_smem(scan_kernel<DKP, T, PS, STORE>, smem);
  if (e != cudaSuccess) return e;
  scan_kernel<DKP, T, PS, STORE><<<grid, 256, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int PS, bool STORE>
cudaError_t pick_scan(const Params& p, cudaStream_t s) {
  return p.dk <= 64 ? run_scan<64, T, PS, STORE>(p, s) : run_scan<128, T, PS, STORE>(p, s);
}

}  // namespace

cudaError_t launch_scan(const Params& p, int dtype, cudaStream_t s) {
  constexpr int B = kBackPieces;
  if (dtype == 1) return p.backward ? pick_scan<__nv_bfloat16, B, true>(p, s) : pick_scan<__nv_bfloat16, 2, false>(p, s);
  if (dtype == 2) return p.backward ? pick_scan<__half, B, true>(p, s) : pick_scan<__half, 2, false>(p, s);
  return p.backward ? pick_scan<float, B, true>(p, s) : pick_scan<float, 3, false>(p, s);
}

}  // namespace delta
}  // namespace qrb
