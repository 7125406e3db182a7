// The backward recurrence of the gated delta rule: the state's gradient walks a sequence's
// chunks from the last to the first (mathematics in qrb_delta.cuh).
//
// As in the forward recurrence a block owns one (sequence, value head, 32-column tile), the
// gradient's tile stays in accumulators and its pieces in shared memory.  Per chunk: K dS' and
// P^T dO give du0, X^T (beta du0) gives du, then Q^T (scale gamma dO) and K^T (-gamma dV) give the
// gradient before the chunk.  dS' and du go to the workspace for the gradients of q and k; the
// sums over value columns that dbeta and dg are made of are taken here, from fp32 accumulators.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

template <int DKP, typename T>
struct RLayout {
  static constexpr int P = Pieces<T>::kIn, PS = kBackPieces;
  static constexpr int PG = Pieces<T>::kS;   // pieces of du and dS' the gradient kernel reads
  static constexpr int kK = tile_bytes(kChunk, P, DKP);
  static constexpr int kX = tile_bytes(kChunk, PS, kChunk);
  static constexpr int kGates = 3 * kChunk * 4;
  static constexpr int kOffQ = kK, kOffX = 2 * kK, kOffP = kOffX + kX, kOffG = kOffP + kX;
  static constexpr int kStage = kOffG + 1024;
  static constexpr int kS = tile_bytes(DKP, PS, kTile);
  static constexpr int kF = tile_bytes(kChunk, PS, kTile);
  static constexpr int kD = tile_bytes(kChunk, P, kTile);
  static constexpr int kStages = 2 * kStage + kS + kD + 2 * kF <= 232448 ? 2 : 1;
  // beta du0 is consumed before -gamma dV is written, behind one more barrier: they share a tile
  static constexpr int kOffS = kStages * kStage, kOffD = kOffS + kS, kOffDS = kOffD + kD, kOffF = kOffDS + kF;
  static constexpr int kBytes = kOffF + kF;
  static_assert(kBytes <= 232448, "shared memory of one block");
};

template <int DKP, typename T>
__global__ void __launch_bounds__(256) rscan_kernel(Params p) {
  using L = RLayout<DKP, T>;
  constexpr int P = L::P, PS = L::PS;
  constexpr int SNT = DKP == 128 ? 4 : 2;
  extern __shared__ __align__(128) unsigned char sm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int tile = blockIdx.x % p.nv, sh = blockIdx.x / p.nv, h = sh % p.hv, seq = sh / p.hv;
  const int hk = h / p.group, n0 = tile * kTile;
  const int sm0 = DKP == 128 ? 16 * warp : 16 * (warp & 3), sn0 = DKP == 128 ? 0 : 16 * (warp >> 2);
  const int m0 = 16 * (warp & 3), c0 = 16 * (warp >> 2);
  unsigned char *S = sm + L::kOffS, *D = sm + L::kOffD, *DS = sm + L::kOffDS, *F = sm + L::kOffF;
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
      st[j][r] = p.ds_end != nullptr && row < p.dk && col < p.dv ? p.ds_end[sbase + (size_t)row * p.dv + col] : 0.f;
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
  if (L::kStages == 2 && nc > 0) load(nc - 1, (nc - 1) & 1);
  for (int c = nc - 1; c >= 0; --c) {
    const int stage = L::kStages == 2 ? (c & 1) : 0;
    unsigned char* d = sm + stage * L::kStage;
    const float* gates = reinterpret_cast<const float*>(d + L::kOffG);
    const int64_t left = n - (int64_t)c * kChunk;
    const int len = left < kChunk ? (int)left : kChunk;
    const int64_t tok = t0 + (int64_t)c * kChunk;
    float v[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = m0 + gr + 8 * (r >> 1), col = n0 + c0 + 8 * j + 2 * tq + (r & 1);
        v[j][r] = row < len && col < p.dv
                      ? to_f(static_cast<const T*>(p.d_o)[b * p.dos.b + (tok + row) * p.dos.t + h * p.dos.h + col])
                      : 0.f;
      }
    if (L::kStages == 2) {
      cp_wait_all();
      __syncthreads();
      if (c > 0) load(c - 1, stage ^ 1);
    } else {
      __syncthreads();
      load(c, 0);
      cp_wait_all();
      __syncthreads();
    }
    const size_t at = slot_head(p, slot0 + c, h) * p.nv + tile;
    {
      unsigned char* to = p.dsp + at * L::kS;
      for (int i = tid * 16; i < tile_bytes(DKP, L::PG, kTile); i += 256 * 16)
        *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(S + i);
    }
    // <S', dS'>: S' is the next chunk's first state, behind the last chunk the final state
    float sds = 0.f;
    {
      const unsigned char* nx = c + 1 < nc ? p.s0p + (slot_head(p, slot0 + c + 1, h) * p.nv + tile) * L::kS : nullptr;
#pragma unroll
      for (int j = 0; j < SNT; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = sm0 + gr + 8 * r, col = sn0 + 8 * j + 2 * tq;
          float2 x = make_float2(0.f, 0.f);
          if (nx != nullptr) {
            x = get2<PS>(nx, DKP, kTile, row, col);
          } else if (row < p.dk) {
            const float* y = p.s_last + sbase + (size_t)row * p.dv + n0 + col;
            if (n0 + col < p.dv) x.x = y[0];
            if (n0 + col + 1 < p.dv) x.y = y[1];
          }
          sds += x.x * st[j][2 * r] + x.y * st[j][2 * r + 1];
        }
    }
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
        const int row = m0 + gr + 8 * r, col = c0 + 8 * j + 2 * tq;
        put2<P>(D, kChunk, kTile, row, col, v[j][2 * r], v[j][2 * r + 1]);
        const float sg = p.scale * gam[r];
        put2<PS>(DS, kChunk, kTile, row, col, sg * v[j][2 * r], sg * v[j][2 * r + 1]);
      }
    float u[2][4];
    zero(u);
    mma_tile<2, false, true, P, PS, PS>(u, d, kChunk, DKP, m0, S, DKP, kTile, c0, 0, DKP);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) u[j][r] *= tail[r >> 1];
    __syncthreads();
    // P^T and X^T are upper triangular: nothing left of this warp's rows
    mma_tile<2, true, true, PS, P, PS>(u, d + L::kOffP, kChunk, kChunk, m0, D, kChunk, kTile, c0, m0, kChunk);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        put2<PS>(F, kChunk, kTile, m0 + gr + 8 * r, c0 + 8 * j + 2 * tq, bet[r] * u[j][2 * r],
                 bet[r] * u[j][2 * r + 1]);
    __syncthreads();
    mma_tile<2, true, true, PS, PS, PS>(u, d + L::kOffX, kChunk, kChunk, m0, F, kChunk, kTile, c0, m0, kChunk);
    __syncthreads();   // F is read before it is written again
    float vdv[2] = {0.f, 0.f}, edu[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = m0 + gr + 8 * r, col = c0 + 8 * j + 2 * tq;
        put2<L::PG>(p.dup + at * L::kF, kChunk, kTile, row, col, u[j][2 * r], u[j][2 * r + 1]);
        const float2 e = get2<PS>(p.ep + at * L::kF, kChunk, kTile, row, col);
        edu[r] += e.x * u[j][2 * r] + e.y * u[j][2 * r + 1];
        const float y0 = bet[r] * u[j][2 * r], y1 = bet[r] * u[j][2 * r + 1];
        put2<PS>(F, kChunk, kTile, row, col, -gam[r] * y0, -gam[r] * y1);
        if (row < len) {
          T* dv = static_cast<T*>(p.dv_) + ((b * p.time + tok + row) * p.hv + h) * p.dv + n0 + col;
          const T* vv = static_cast<const T*>(p.v) + b * p.vs.b + (tok + row) * p.vs.t + h * p.vs.h + n0 + col;
          if (n0 + col < p.dv) {
            dv[0] = from_f<T>(y0);
            vdv[r] += to_f(vv[0]) * y0;
          }
          if (n0 + col + 1 < p.dv) {
            dv[1] = from_f<T>(y1);
            vdv[r] += to_f(vv[1]) * y1;
          }
        }
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        vdv[r] += __shfl_xor_sync(0xffffffffu, vdv[r], o);
        edu[r] += __shfl_xor_sync(0xffffffffu, edu[r], o);
      }
      if (tq == 0) {
        p.vdv[(at * 2 + (warp >> 2)) * kChunk + m0 + gr + 8 * r] = vdv[r];
        p.edu[(at * 2 + (warp >> 2)) * kChunk + m0 + gr + 8 * r] = edu[r];
      }
    }
    sds = warp_sum(sds);
    if (lane == 0) p.sds[at * 8 + warp] = sds;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SNT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[j][r] *= glast;
    mma_tile<SNT, true, true, P, PS, PS>(st, d + L::kOffQ, kChunk, DKP, sm0, DS, kChunk, kTile, sn0, 0, kChunk);
    mma_tile<SNT, true, true, P, PS, PS>(st, d, kChunk, DKP, sm0, F, kChunk, kTile, sn0, 0, kChunk);
    put_state();
  }
  if (p.ds_init != nullptr) {
#pragma unroll
    for (int j = 0; j < SNT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = sm0 + gr + 8 * (r >> 1), col = n0 + sn0 + 8 * j + 2 * tq + (r & 1);
        if (row < p.dk && col < p.dv) p.ds_init[sbase + (size_t)row * p.dv + col] = st[j][r];
      }
  }
}

template <int DKP, typename T>
cudaError_t run_rscan(const Params& p, cudaStream_t s) {
  constexpr int smem = RLayout<DKP, T>::kBytes;
  const double rows = (double)p.bound * kChunk * p.hv;
  LaunchTimer t("delta_rscan_kernel", s, rows * 2.0 * p.dv * sizeof(T), rows * 6.0 * p.dk * p.dv);
  cudaError_t e = allow_smem(rscan_kernel<DKP, T>, smem);
  if (e != cudaSuccess) return e;
  rscan_kernel<DKP, T><<<(unsigned)p.nseq * p.hv * p.nv, 256, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rscan(const Params& p, int dtype, cudaStream_t s) {
  if (dtype == 1) return p.dk <= 64 ? run_rscan<64, __nv_bfloat16>(p, s) : run_rscan<128, __nv_bfloat16>(p, s);
  if (dtype == 2) return p.dk <= 64 ? run_rscan<64, __half>(p, s) : run_rscan<128, __half>(p, s);
  return p.dk <= 64 ? run_rscan<64, float>(p, s) : run_rscan<128, float>(p, s);
}

}  // namespace delta
}  // namespace qrb
