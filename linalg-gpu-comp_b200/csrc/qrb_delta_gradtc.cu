// Gradients of q and k (and the sums of g's and beta's) for 16-bit inputs, on the tensor cores through
// tcgen05; qrb_delta_grad.cu has fp32 and the mathematics in words.
//
// The transposed gradients are formed, tensor-memory lane = q/k column, so that S0, dS', K and Q are A
// operands of 128 rows in the layouts they were written in, with value columns (or tokens) along k:
//     [aq | ay]^T = S0 [dO | du]^T        au^T = dS' e^T        [az ; an] = [dO ; du] e
//     dq^T = scale gam aq^T + K^T Z^T     dk^T = tail bet au^T - gam bet ay^T + Q^T Z + K^T (N + N^T)
// with Z, N the masked and decayed az, an.
// For dk up to 64 the rows are S0's and dS's, K's and Q's side by side: half of what is computed is not
// read, and the upper half of the lanes hands its part of dk to the lower one through shared memory.
// Two pieces of S0, dS', e, du, Z, N leave 2^-18 of each, far
// below the 16-bit outputs.  A block walks over (chunk, q/k head) pairs: one thread loads value tiles of 32
// columns into a ring, one issues the products, sixteen warps scale and store, and one warp adds up dg and
// dbeta.  Heads of a group are added in order, in registers.
// It reads 240 KB a chunk and value head (dk = dv = 128, bf16), which bounds it: 2048 of them in 120 us, 4.1
// TB/s, with three tiles of 52 KB in flight an SM.
#include "qrb_delta_tc.cuh"

namespace qrb {
namespace delta {
namespace {

constexpr int kGateWarp = kLoader + 1, kGradThreads = 32 * (kGateWarp + 1);

template <int DKP, typename T>
struct TLayout {
  static constexpr bool kHalf = DKP == 64;   // S0 and dS', K and Q share the 128 rows
  static constexpr int P = Pieces<T>::kIn, PS = 2;
  static constexpr int kStages = kHalf ? (P == 1 ? 4 : 3) : (P == 1 ? 3 : 2);
  static constexpr int kT = kTile * kChunk * 2, kS = kTile * DKP * 2;   // a piece of a token tile, of a state tile
  static constexpr int kWS = tile_bytes(kTile, kBackPieces, DKP), kWF = tile_bytes(kTile, kBackPieces, kChunk);
  // First pieces dO | du, then (dk above 64) second pieces, e, S0 and dS' with both pieces each; or e, second
  // pieces with e's, and [S0 | dS'] a piece.  Second pieces: du', and dO' before it where there is one, so
  // that [dO ; du] lie together and so do [dO' ; du'].
  static constexpr int kOffDU = kT, kOffE = kHalf ? 2 * kT : (P + 2) * kT;
  static constexpr int kOffLo = kHalf ? 3 * kT : 2 * kT, kOffDULo = kOffLo + (P - 1) * kT;
  static constexpr int kOffELo = kHalf ? kOffDULo + kT : kOffE + kT;
  static constexpr int kOffS = kOffELo + kT, kOffDS = kHalf ? kOffS + kS : kOffS + 2 * kS;
  static constexpr int kStep = kHalf ? 2 * kS : kS;   // between pieces of S0 and of dS'
  static constexpr int kStage = kOffS + 4 * kS;
  static constexpr int kK = tile_bytes(kChunk, P, DKP), kZ = tile_bytes(kChunk, PS, kChunk);
  static constexpr int kOffK = kStages * kStage, kOffQ = kOffK + kK, kOffZ = kOffQ + kK, kOffN = kOffZ + kZ;
  static constexpr int kOffX = kOffN + kZ;   // kHalf: what the upper lanes hold of dk
  static constexpr int kBar = kOffX + (kHalf ? kChunk * 64 * 4 : 0);
  static constexpr int kBytes = kBar + 256 + 1024;   // 1024: alignment
  static_assert(kBytes <= kSmemLimit && kStage % 1024 == 0, "shared memory of one block");
  // tensor memory columns: [aq | ay], au | [az ; an] | their second pieces of dO, du | dq | dk | kHalf: dk of N
  static constexpr uint32_t tA = 0, tU = 128, tZ = 192, tLo = 256, tDQ = 320, tDK = 384, tDN = kHalf ? 448 : 384;
};

struct GradBars {
  uint64_t full[4], empty[4], kq, acc, zn, read, done, over, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(GradBars) <= 256, "barrier block");

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// Sixteen values as two pieces in row `row` of a swizzled tile of 64 columns a piece.
__device__ __forceinline__ void put_row(unsigned char* tile, int row, int col, float (&x)[kTok]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[kTok / 2];
#pragma unroll
    for (int j = 0; j < kTok / 2; ++j) {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(x[2 * j + 1]), "f"(x[2 * j]));
      x[2 * j] -= __uint_as_float(w[j] << 16);
      x[2 * j + 1] -= __uint_as_float(w[j] & 0xffff0000u);
    }
#pragma unroll
    for (int j = 0; j < kTok / 2; j += 4)
      *reinterpret_cast<uint4*>(tile + tile_off(kChunk, row, i * kChunk + col + 2 * j)) =
          make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
  }
}

template <int DKP, typename T>
__global__ void __launch_bounds__(kGradThreads, 1) grad_tc_kernel(const __grid_constant__ Params p, int* err) {
  using L = TLayout<DKP, T>;
  constexpr int P = L::P;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                       ~uintptr_t(1023));
  GradBars& bars = *reinterpret_cast<GradBars*>(sm + L::kBar);
  volatile int* abort = &bars.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t items = (int64_t)p.bound * p.hk;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    for (uint64_t* x : {&bars.kq, &bars.acc, &bars.done, &bars.drain}) mbar_init(x, 1);
    for (uint64_t* x : {&bars.zn, &bars.read}) mbar_init(x, 4 * kParts);
    mbar_init(&bars.over, 2 * kParts);
    bars.abort = 0;
    fence_mbar_init();
  }
  if (warp == kIssuer) tmem_alloc(&bars.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  // every role walks over the same (chunk, q/k head) pairs; packed layouts have chunk slots without a chunk
  auto next = [&](int64_t i) {
    do i += gridDim.x;
    while (i < items && p.offsets != nullptr && i / p.hk >= p.cstart[p.nseq]);
    return i;
  };
  const int64_t first = next((int64_t)blockIdx.x - gridDim.x);

  if (warp == kLoader) {
    // ---------------- loads: one thread ----------------
    if (lane == 0) {
      uint32_t tiles = 0, unit = 0, pairs = 0;
      bool ok = true;
      for (int64_t i = first; i < items && ok; i = next(i)) {
        const int c = (int)(i / p.hk), hk = (int)(i - (int64_t)c * p.hk);
        for (int hh = 0; hh < p.group && ok; ++hh, ++unit) {
          const size_t at = slot_head(p, c, hk * p.group + hh) * p.nv;
          for (int n = 0; n < p.nv; ++n, ++tiles) {
            const uint32_t stage = tiles % L::kStages;
            if (tiles >= L::kStages &&
                !(ok = mbar_wait_abort(&bars.empty[stage], (tiles / L::kStages - 1) & 1, abort, err, 91)))
              break;
            // Once a unit, in order, and before its last tile, so that this unit's own products cannot be done (a
            // wait by parity tells a phase from its neighbours only): the last one's are.  K and Q, which go
            // where the last pair's lay, could not come earlier; the tiles before this one could.
            if (n == min(p.nv, L::kStages) - 1) {
              if (unit > 0 && !(ok = mbar_wait_abort(&bars.done, (unit - 1) & 1, abort, err, 92))) break;
              if (hh == 0) {
                const size_t qk = ((size_t)c * p.hk + hk) * L::kK;
                mbar_arrive_expect_tx(&bars.kq, 2 * L::kK);
                bulk_load(sm + L::kOffK, p.kt + qk, L::kK, &bars.kq);
                bulk_load(sm + L::kOffQ, p.qt + qk, L::kK, &bars.kq);
                ++pairs;
              }
            }
            unsigned char* d = sm + stage * L::kStage;
            uint64_t* bar = &bars.full[stage];
            const unsigned char *o = p.dop + (at + n) * P * L::kT, *u = p.dup + (at + n) * L::kWF;
            mbar_arrive_expect_tx(bar, L::kStage);
            const unsigned char *e = p.ep + (at + n) * L::kWF, *s0 = p.s0p + (at + n) * L::kWS,
                                *ds = p.dsp + (at + n) * L::kWS;
            bulk_load(d, o, L::kT, bar);
            if (P > 1) bulk_load(d + L::kOffLo, o + L::kT, L::kT, bar);
            if (L::kOffDULo == L::kOffDU + L::kT) {
              bulk_load(d + L::kOffDU, u, 2 * L::kT, bar);
            } else {
              bulk_load(d + L::kOffDU, u, L::kT, bar);
              bulk_load(d + L::kOffDULo, u + L::kT, L::kT, bar);
            }
            if (L::kHalf) {
              bulk_load(d + L::kOffE, e, L::kT, bar);
              bulk_load(d + L::kOffELo, e + L::kT, L::kT, bar);
              for (int i = 0; i < 2; ++i) {
                bulk_load(d + L::kOffS + i * L::kStep, s0 + i * L::kS, L::kS, bar);
                bulk_load(d + L::kOffDS + i * L::kStep, ds + i * L::kS, L::kS, bar);
              }
            } else {
              bulk_load(d + L::kOffE, e, 2 * L::kT, bar);
              bulk_load(d + L::kOffS, s0, 2 * L::kS, bar);
              bulk_load(d + L::kOffDS, ds, 2 * L::kS, bar);
            }
          }
        }
      }
      if (*abort) {   // loads in flight must land before the block's memory goes
        for (uint32_t i = 0; i < L::kStages; ++i)
          if (tiles > i) mbar_wait(&bars.full[i], ((tiles - 1 - i) / L::kStages) & 1, 1u << 22);
        if (pairs > 0) mbar_wait(&bars.kq, (pairs - 1) & 1, 1u << 22);
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    // ---------------- products: one thread ----------------
    if (lane == 0) {
      constexpr uint32_t kAmn = 1u << 15;
      constexpr uint32_t all = idesc_bf16(192, 1) | kAmn, wide = idesc_bf16(128, 1) | kAmn;
      constexpr uint32_t mn = idesc_bf16(64, 1) | kAmn, km = idesc_bf16(64, 0) | kAmn;
      // tiles of the recurrences: 16-byte units of 8 columns, 32 value rows apart; 16 rows a step
      auto unitd = [](uint32_t a, int k) { return sdesc_make(a + 256u * k, 128, kTile * 16, 0); };
      // K, Q: columns as M (K's 128, or K's 64 and Q's); Z, N: rows (tokens) as N or across them; 16 tokens a step
      auto across = [](uint32_t a, int k) {
        return sdesc_sw128(a + 2048u * k, L::kHalf ? L::kK : kChunk * 128, 1024);
      };
      auto along = [](uint32_t a, int k) { return sdesc_sw128(a + 32u * k, 16, 1024); };
      const uint32_t base = smem_u32(sm);
      uint32_t tiles = 0, unit = 0, item = 0;
      bool ok = true;
      for (int64_t i = first; i < items && ok; i = next(i), ++item)
        for (int hh = 0; hh < p.group && ok; ++hh, ++unit) {
          if (unit > 0 && !(ok = mbar_wait_abort(&bars.read, (unit - 1) & 1, abort, err, 93))) break;
          for (int n = 0; n < p.nv; ++n, ++tiles) {
            const uint32_t stage = tiles % L::kStages;
            if (!(ok = mbar_wait_abort(&bars.full[stage], (tiles / L::kStages) & 1, abort, err, 94))) break;
            tc_fence_after();
            const uint32_t d = base + stage * L::kStage, lo = d + L::kOffLo, dul = d + L::kOffDULo, e = d + L::kOffE,
                           el = d + L::kOffELo, s = d + L::kOffS, ds = d + L::kOffDS;
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k) {
              const uint32_t acc = n > 0 || k > 0;
              if (L::kHalf) {   // [S0 ; dS'] [dO | du | e]
                mma_ss(tmem + L::tA, unitd(s + L::kStep, k), unitd(d, k), all, acc);
                mma_ss(tmem + L::tA, unitd(s, k), unitd(d, k), all, 1);
                if (P > 1) mma_ss(tmem + L::tA, unitd(s, k), unitd(lo, k), all, 1);
                else mma_ss(tmem + L::tA + 64, unitd(s, k), unitd(dul, k), wide, 1);
              } else {
                mma_ss(tmem + L::tA, unitd(s + L::kStep, k), unitd(d, k), wide, acc);
                mma_ss(tmem + L::tA, unitd(s, k), unitd(d, k), wide, 1);
                mma_ss(tmem + L::tA + 64, unitd(s, k), unitd(dul, k), mn, 1);
                if (P > 1) mma_ss(tmem + L::tA, unitd(s, k), unitd(lo, k), mn, 1);
                mma_ss(tmem + L::tU, unitd(ds + L::kStep, k), unitd(e, k), mn, acc);
                mma_ss(tmem + L::tU, unitd(ds, k), unitd(el, k), mn, 1);
                mma_ss(tmem + L::tU, unitd(ds, k), unitd(e, k), mn, 1);
              }
              mma_ss(tmem + L::tZ, unitd(d, k), unitd(el, k), mn, acc);
              mma_ss(tmem + L::tZ, unitd(d, k), unitd(e, k), mn, 1);
              // the lower half du', the upper one dO' or, with one piece, nothing that is read
              mma_ss(tmem + L::tLo, unitd(dul - L::kT, k), unitd(e, k), mn, acc);
            }
            mma_commit(&bars.empty[stage]);
          }
          if (!ok) break;
          mma_commit(&bars.acc);
          if (!(ok = mbar_wait_abort(&bars.zn, unit & 1, abort, err, 95))) break;
          if (hh == 0 && !(ok = mbar_wait_abort(&bars.kq, item & 1, abort, err, 96))) break;
          tc_fence_after();
          const uint32_t K = base + L::kOffK, Z = base + L::kOffZ, N = base + L::kOffN;
          constexpr uint32_t kZp = kChunk * 128, kKp = kChunk * 2 * DKP;   // a piece of Z or N, of K or Q
#pragma unroll
          for (int w = 1; w >= 0; --w)
#pragma unroll
            for (int a = 0; a < P; ++a) {
              const int z = w - a;   // pieces a + z = w
              if (z < 0) continue;
#pragma unroll
              for (int k = 0; k < kChunk / 16; ++k) {
                const uint32_t acc = !(w == 1 && a == 0 && k == 0);
                const uint64_t ka = across(K + a * kKp, k), qa = L::kHalf ? ka : across(K + L::kK + a * kKp, k);
                // across of Z and N: one block of 64 columns, so that the distance between blocks is not used
                mma_ss(tmem + L::tDQ, ka, along(Z + z * kZp, k), km, acc);
                mma_ss(tmem + L::tDK, qa, across(Z + z * kZp, k), mn, acc);
                mma_ss(tmem + L::tDN, ka, along(N + z * kZp, k), km, L::kHalf ? acc : 1);
                mma_ss(tmem + L::tDN, ka, across(N + z * kZp, k), mn, 1);
              }
            }
          mma_commit(&bars.done);
        }
      if (*abort) {   // MMAs in flight must end before tensor memory goes
        mma_commit(&bars.drain);
        mbar_wait(&bars.drain, 0, 1u << 22);
      }
    }
    __syncwarp();
  } else if (warp == kGateWarp) {
    // ---------------- dbeta, dg: two tokens a lane ----------------
    for (int64_t i = first; i < items; i = next(i)) {
      const int c = (int)(i / p.hk), hk = (int)(i - (int64_t)c * p.hk);
      const Chunk ch = chunk_at(p, c);
      for (int hh = 0; hh < p.group; ++hh) gate_sums(p, ch, slot_head(p, c, hk * p.group + hh), hk * p.group + hh, lane);
    }
  } else {
    // ---------------- scaling and stores ----------------
    const int q = warp & 3, part = warp >> 2, tb = kTok * part;
    const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16) + tb;
    // q/k column; kHalf: the upper lanes (K's and dS's products lie in them) hand over what they have of dk
    const bool upper = L::kHalf && q >= 2;
    const int col = (32 * q + lane) & (DKP - 1);
    const int row = (32 * q + lane) & (kChunk - 1);   // token of az (the first half of the lanes) and an
    uint32_t unit = 0;
    bool ok = true;
    for (int64_t i = first; i < items && ok; i = next(i)) {
      const int c = (int)(i / p.hk), hk = (int)(i - (int64_t)c * p.hk);
      float dq[kTok], dk[kTok];
#pragma unroll
      for (int j = 0; j < kTok; ++j) dq[j] = dk[j] = 0.f;
      for (int hh = 0; hh < p.group; ++hh, ++unit) {
        const size_t at = slot_head(p, c, hk * p.group + hh);
        const float* gates = p.gates + at * 3 * kChunk;
        float f[kTok], x[kTok];
        const int last = q < 2 ? row : row - 1;   // Z has its diagonal, N has not
        {
          const double* G = p.gsum + at * kChunk;
          const double gi = __ldg(G + row);
          const float mine = q < 2 ? p.scale : -__ldg(gates + 2 * kChunk + row);
#pragma unroll
          for (int j = 0; j < kTok; ++j) {
            const float d = expf((float)(gi - __ldg(G + tb + j))) * __ldg(gates + 2 * kChunk + tb + j) * mine;
            f[j] = tb + j <= last ? d : 0.f;
          }
        }
        if (!(ok = warp_wait(&bars.acc, unit & 1, abort, err, 97))) break;
        tc_fence_after();
        ld_cols(tl + L::tZ, x);
        if (P > 1 || q >= 2) {
          float y[kTok];
          ld_cols(tl + L::tLo, y);
#pragma unroll
          for (int j = 0; j < kTok; ++j) x[j] += y[j];
        }
#pragma unroll
        for (int j = 0; j < kTok; ++j) x[j] = tb + j <= last ? f[j] * x[j] : 0.f;
        put_row(sm + (q < 2 ? L::kOffZ : L::kOffN), row, tb, x);
        fence_proxy_async();
        tc_fence_before();
        warp_arrive(&bars.zn);
        const float4 *gam = reinterpret_cast<const float4*>(gates + tb), *tail = gam + kChunk / 4, *bet = tail + kChunk / 4;
        float* over = reinterpret_cast<float*>(sm + L::kOffX) + tb * 64 + col;
        if (!upper) {
          ld_cols(tl + L::tA, x);
          with_tokens(gam, [&](int j, float g) { dq[j] += p.scale * g * x[j]; });
          ld_cols(tl + L::tA + 64, x);
          with_tokens(gam, [&](int j, float g) { x[j] *= -g; });
        } else {
#pragma unroll
          for (int j = 0; j < kTok; ++j) x[j] = 0.f;
        }
        if (!L::kHalf || upper) {
          ld_cols(tl + L::tU, f);
          with_tokens(tail, [&](int j, float g) { x[j] += g * f[j]; });
        }
        with_tokens(bet, [&](int j, float g) { x[j] *= g; });
        tc_fence_before();
        warp_arrive(&bars.read);
        if (!(ok = warp_wait(&bars.done, unit & 1, abort, err, 98))) break;
        tc_fence_after();
        if (upper) {
          ld_cols(tl + L::tDK, f);
#pragma unroll
          for (int j = 0; j < kTok; ++j) over[j * 64] = x[j] + f[j];
          warp_arrive(&bars.over);
        } else {
          ld_cols(tl + L::tDN, f);
#pragma unroll
          for (int j = 0; j < kTok; ++j) dk[j] += x[j] + f[j];
          ld_cols(tl + L::tDQ, x);
#pragma unroll
          for (int j = 0; j < kTok; ++j) dq[j] += x[j];
          if (L::kHalf) {
            if (!(ok = warp_wait(&bars.over, unit & 1, abort, err, 99))) break;
#pragma unroll
            for (int j = 0; j < kTok; ++j) dk[j] += over[j * 64];
          }
        }
        tc_fence_before();
      }
      if (!ok) break;
      if (!upper && col < p.dk) {
        const Chunk ch = chunk_at(p, c);
        const size_t to = ((size_t)(ch.b * p.time + ch.t0 + tb) * p.hk + hk) * p.dk + col;
        const int64_t stride = (int64_t)p.hk * p.dk;
        store_tokens(static_cast<T*>(p.dq) + to, stride, ch.len - tb, dq);
        store_tokens(static_cast<T*>(p.dk_) + to, stride, ch.len - tb, dk);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

template <int DKP, typename T>
cudaError_t run_grad_tc(const Params& p, cudaStream_t s) {
  constexpr int smem = TLayout<DKP, T>::kBytes;
  const double rows = (double)p.bound * kChunk * p.hv;
  int* err = device_error_flag();
  if (err == nullptr) return cudaErrorInvalidValue;
  LaunchTimer t("delta_grad_tc_kernel", s, rows * 4.0 * p.dk * sizeof(T), rows * (6.0 * p.dv + 8.0 * kChunk) * p.dk);
  cudaError_t e = allow_smem<grad_tc_kernel<DKP, T>>(smem);
  if (e != cudaSuccess) return e;
  const int64_t items = (int64_t)p.bound * p.hk;
  grad_tc_kernel<DKP, T><<<(unsigned)(items < sm_count() ? items : sm_count()), kGradThreads, smem, s>>>(p, err);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_grad_tc(const Params& p, cudaStream_t s) {
  return p.dk <= 64 ? run_grad_tc<64, T>(p, s) : run_grad_tc<128, T>(p, s);
}
template cudaError_t launch_grad_tc<__nv_bfloat16>(const Params&, cudaStream_t);
template cudaError_t launch_grad_tc<__half>(const Params&, cudaStream_t);

}  // namespace delta
}  // namespace qrb
