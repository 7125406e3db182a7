// The backward recurrence of the gated delta rule: the state's gradient walks a sequence's chunks
// from the last to the first (mathematics in qrb_delta.cuh, data flow in qrb_delta_tc.cuh).
//
// As in the forward recurrence a block owns one (sequence, value head, up to 128 value columns), a
// thread a quarter of a column of the gradient.  Per chunk, transposed (lane = value column):
//     K dS' -> du0 = tail (K dS') + P^T dO, F = beta du0 -> X^T F -> du = du0 + X^T F, dV = beta du
//     -> Q^T (scale gamma dO) + K^T (-gamma dV) -> dS = gamma_last dS' + ...
// P^T dO and Q^T (...) run in the shadow of the register work.  dS' and du go to the workspace for
// the gradients of q and k; the sums over value columns that dbeta and dg are made of are taken here,
// from fp32 values: e.du, v.dV per token and <S', dS'> per chunk.
// Measured (dk = dv = 128, bf16, 128 blocks at once): 12.3 us a chunk, 336 KB at 3.5 TB/s; the state alone
// takes 6.3.
#include "qrb_delta_tc.cuh"
#include "qrb_ring.cuh"

namespace qrb {
namespace delta {
namespace {

template <int DKP, typename T>
struct RLayout {
  static constexpr int P = Pieces<T>::kIn, PS = kBackPieces;
  static constexpr int PG = Pieces<T>::kS;   // pieces of du and dS' the gradient kernel reads
  static constexpr int kK = tile_bytes(kChunk, P, DKP);
  static constexpr int kX = tile_bytes(kChunk, PS, kChunk);
  static constexpr int kV = kChunk * kLanes * (int)sizeof(T);
  static constexpr int kGates = 3 * kChunk * 4;
  static constexpr int kOffQ = kK, kOffX = 2 * kK, kOffP = kOffX + kX, kOffV = kOffP + kX, kOffD = kOffV + kV;
  static constexpr int kStage = kOffD + kV;
  static constexpr int kStages = 2 * (kStage + kGates) + 256 + 1024 <= kSmemLimit ? 2 : 1;
  static constexpr int kOffG = kStages * kStage;
  static constexpr int kBar = kOffG + kStages * kGates;
  static constexpr int kBytes = kBar + 256 + 1024;
  static_assert(kBytes <= kSmemLimit, "shared memory of one block");
  // tensor memory: pieces of dS', then the sum of K^T and Q^T products over them | K dS', then X^T F
  // | P^T dO | scale gamma dO | dO, then F, then -gamma dV
  static constexpr uint32_t kSp = PS * (DKP / 2);
  static constexpr uint32_t tS = 0, tD = 0, tK = kSp > (uint32_t)DKP ? kSp : DKP, tP = tK + 64, tO = tP + 64,
                            tF = tO + 32 * PS;
  static_assert(tF + 32 * PS <= 512 && P <= PS, "tensor memory");
};

struct RBars {
  uint64_t full[2], empty[2], sp, dop, ks, pd, f, xf, uw, ds, share[4], drain;   // full, empty: see qrb_ring.cuh
  uint32_t tmem;
  int abort;
  Span span;   // here, not in registers that the loops need
};
static_assert(sizeof(RBars) <= 256, "barrier block");

// STATE: only the gradient of the state, of every segment but a sequence's first: from the final state's
// gradient for the last, else from zero.  It runs beside scan's state-only pass, launched just before it.
template <int DKP, typename T, bool STATE>
__global__ void __launch_bounds__(kTcThreads, 1) rscan_kernel(const __grid_constant__ Params p, int* err) {
  using L = RLayout<DKP, T>;
  using R = Ring<L::kStages>;
  constexpr int P = L::P, PS = L::PS, PG = L::PG, HK = DKP / kParts;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                       ~uintptr_t(1023));
  RBars& bars = *reinterpret_cast<RBars*>(sm + L::kBar);
  volatile int* abort = &bars.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nb = (p.dv + kLanes - 1) / kLanes;
  const int vb = blockIdx.x % nb, sh = blockIdx.x / nb, h = sh % p.hv;
  const Span mine = span_at(p, sh / p.hv);
  if (mine.nc < 0 || (STATE && mine.first)) return;   // (with no other blocks, scan's pass had none either)
  const int hk = h / p.group, nc = mine.nc, slot0 = mine.slot0;
  const int quarters = min(4, (p.dv - vb * kLanes + 31) / 32);

  if (tid == 0) {
    mbar_init(&bars.full[0], 1);
    mbar_init(&bars.full[1], 1);
    for (uint64_t* x : {&bars.ks, &bars.pd, &bars.xf, &bars.ds, &bars.drain}) mbar_init(x, 1);
    for (uint64_t* x : {&bars.sp, &bars.dop, &bars.f, &bars.uw, &bars.empty[0], &bars.empty[1]})
      mbar_init(x, kParts * quarters);
    for (int i = 0; i < 4; ++i) mbar_init(&bars.share[i], kParts);
    bars.abort = 0;
    bars.span = mine;
    fence_mbar_init();
  }
  if (warp == kIssuer) tmem_alloc(&bars.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;

  if (warp == kLoader) {
    // ---------------- loads: one thread; step i handles chunk nc - 1 - i ----------------
    if (lane == 0) {
      int i = 0;
      for (; i < nc; ++i) {
        const int stage = R::stage(i), c = nc - 1 - i;
        if (i >= L::kStages && !mbar_wait_abort(&bars.empty[stage], R::phase(i - L::kStages), abort, err, 71)) break;
        unsigned char* d = sm + stage * L::kStage;
        uint64_t* bar = &bars.full[stage];
        const size_t qk = ((size_t)(slot0 + c) * p.hk + hk) * L::kK, at = slot_head(p, slot0 + c, h);
        mbar_arrive_expect_tx(bar, L::kStage + L::kGates);
        bulk_load(d, p.kt + qk, L::kK, bar);
        bulk_load(sm + L::kOffG + stage * L::kGates, p.gates + at * 3 * kChunk, L::kGates, bar);
        bulk_load(d + L::kOffD, p.dot + (at * nb + vb) * L::kV, L::kV, bar);
        bulk_load(d + L::kOffP, p.pt + at * L::kX, L::kX, bar);
        bulk_load(d + L::kOffX, p.xt + at * L::kX, L::kX, bar);
        bulk_load(d + L::kOffQ, p.qt + qk, L::kK, bar);
        bulk_load(d + L::kOffV, p.vt + (at * nb + vb) * L::kV, L::kV, bar);
        if (!STATE) {   // what the sums of this chunk will read
          constexpr int kWS = tile_bytes(kTile, PS, DKP), kWF = tile_bytes(kTile, PS, kChunk);
          bulk_prefetch(p.ep + (at * p.nv + 4 * vb) * kWF, quarters * kWF);
          bulk_prefetch(p.odo + (at * p.nv + 4 * vb) * kChunk, quarters * kChunk * 4);
          if (i > 0 && i % kAnchor == 0)
            bulk_prefetch(p.s0p + (slot_head(p, slot0 + c + 1, h) * p.nv + 4 * vb) * kWS, quarters * kWS);
        }
      }
      if (*abort)   // loads in flight must land before the block's memory goes
        for (int s = 0; s < L::kStages; ++s)
          if (i > s) mbar_wait(&bars.full[s], R::phase(i - 1 - s), 1u << 22);
    }
  } else if (warp == kIssuer) {
    // ---------------- MMAs: one thread ----------------
    if (lane == 0) {
      for (int i = 0; i < nc; ++i) {
        const uint32_t ph = i & 1, sb = smem_u32(sm + R::stage(i) * L::kStage);
        if (!mbar_wait_abort(&bars.full[R::stage(i)], R::phase(i), abort, err, 72)) break;
        if (!mbar_wait_abort(&bars.sp, ph, abort, err, 73)) break;
        tc_fence_after();
        mma_pieces<64, DKP, false, PS, P, PS>(tmem + L::tK, tmem + L::tS, DKP / 2, sb, 0);
        mma_commit(&bars.ks);
        if (!mbar_wait_abort(&bars.dop, ph, abort, err, 75)) break;
        tc_fence_after();
        mma_pieces<64, 64, true, P, PS, PS>(tmem + L::tP, tmem + L::tF, 32, sb + L::kOffP, 0);
        mma_commit(&bars.pd);
        if (!mbar_wait_abort(&bars.f, ph, abort, err, 76)) break;
        tc_fence_after();
        mma_pieces<64, 64, true, PS, PS, PS>(tmem + L::tK, tmem + L::tF, 32, sb + L::kOffX, 0);
        mma_commit(&bars.xf);
        mma_pieces<DKP, 64, true, PS, P, PS>(tmem + L::tD, tmem + L::tO, 32, sb + L::kOffQ, 0);
        if (!mbar_wait_abort(&bars.uw, ph, abort, err, 77)) break;
        tc_fence_after();
        mma_pieces<DKP, 64, true, PS, P, PS>(tmem + L::tD, tmem + L::tF, 32, sb, 1);
        mma_commit(&bars.ds);
      }
      if (*abort) {   // MMAs in flight must end before tensor memory goes
        mma_commit(&bars.drain);
        mbar_wait(&bars.drain, 0, 1u << 22);
      }
    }
  } else {
    const Span& span = bars.span;
    const int q = warp & 3, part = warp >> 2;
    if (q < quarters) {
      const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
      const int lcol = 32 * q + lane, col = vb * kLanes + lcol;
      const int tile = vb * 4 + q;
      const int tb = kTok * part, kb = HK * part;
      const bool on = col < p.dv;
      auto sbase = [&] { return (((size_t)span.seq * p.hv + h) * p.dk + kb) * p.dv; };
      const int pitch = nb * kLanes;   // at the borders of segments, as in scan
      auto border = [&](float* x, int g) { return x + (((size_t)g * p.hv + h) * DKP + kb) * pitch + col; };
      constexpr int kWS = tile_bytes(kTile, PS, DKP), kWF = tile_bytes(kTile, PS, kChunk);
      float st[HK];
      if (!STATE && !(span.first && span.last)) {
        load_column(border(p.seg_ds, span.last ? span.g0 : span.g + 1), pitch, HK, true, st);
      } else if (span.last && p.ds_end != nullptr) {
        load_column(p.ds_end + sbase() + min(col, p.dv - 1), p.dv, p.dk - kb, on, st);
      } else {
#pragma unroll
        for (int j = 0; j < HK; ++j) st[j] = 0.f;
      }
      if (STATE && span.last) store_column(border(p.seg_ds, span.g0), pitch, HK, st);
      // pieces of dS' for the products, the first PG of them for the gradient kernel too
      auto put_state = [&](int c) {
        float y[HK];
#pragma unroll
        for (int i = 0; i < HK; ++i) y[i] = st[i];
        unsigned char* to = p.dsp + (slot_head(p, slot0 + c, h) * p.nv + tile) * kWS;
        put_pieces<PS, STATE ? 0 : PG>(tl + L::tS + kb / 2, DKP / 2, y, to, lane, DKP, kb);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&bars.sp);
      };
      float sds = 0.f;
      if (nc > 0) put_state(nc - 1);
      for (int i = 0; i < nc; ++i) {
        const uint32_t ph = i & 1;
        const int c = nc - 1 - i;
        const size_t at = slot_head(p, slot0 + c, h) * p.nv + tile;
        const unsigned char* stage = sm + R::stage(i) * L::kStage;
        const Gates gates(sm + L::kOffG + R::stage(i) * L::kGates, tb);
        float x[kTok], u[kTok];
        if (!warp_wait(&bars.full[R::stage(i)], R::phase(i), abort, err, 81)) break;
        staged<T>(stage + L::kOffD, tb, lcol, x);
        with_tokens(gates.gam, [&](int j, float g) { u[j] = x[j] * (p.scale * g); });
        // (for the gradient kernel too, where it takes them as tiles)
        constexpr int keep = !STATE && grad_on_tc(sizeof(T) == 2) ? P : 0;
        put_pieces<P, keep>(tl + L::tF + tb / 2, 32, x, p.dop + at * tile_bytes(kTile, P, kChunk), lane, kChunk, tb);
        put_pieces<PS, 0>(tl + L::tO + tb / 2, 32, u);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&bars.dop);
        if (!STATE) {
          // This warp's share of <S', dS'>: behind the last chunk from the state there, at every kAnchor-th
          // chunk before it from the next chunk's first state, and between from the next chunk's share, as
          // <S0, dS0> = <S', dS'> + sum (o.do - v.dV) over a chunk's tokens.
          if (i % kAnchor == 0) {
            float y[HK];
            if (i > 0)
              fetch_pieces<PS, HK>(p.s0p + (slot_head(p, slot0 + c + 1, h) * p.nv + tile) * kWS, lane, DKP, kb, y);
            else if (!span.last)
              load_column(border(p.seg_s, span.g + 1), pitch, HK, true, y);
            else
              load_column(p.s_last + sbase() + min(col, p.dv - 1), p.dv, p.dk - kb, on, y);
            sds = 0.f;
#pragma unroll
            for (int a = 0; a < HK; ++a) sds += y[a] * st[a];
            sds = warp_sum(sds);
          }
          if (lane == 0) p.sds[at * kParts + part] = sds;
        }
        if (!warp_wait(&bars.ks, ph, abort, err, 82)) break;
        tc_fence_after();
        ld_cols(tl + L::tK + tb, u);
        with_tokens(gates.tail, [&](int j, float g) { u[j] *= g; });
        if (!warp_wait(&bars.pd, ph, abort, err, 83)) break;
        tc_fence_after();
        ld_cols(tl + L::tP + tb, x);
#pragma unroll
        for (int j = 0; j < kTok; ++j) u[j] += x[j];
        with_tokens(gates.bet, [&](int j, float g) { x[j] = g * u[j]; });
        put_pieces<PS, 0>(tl + L::tF + tb / 2, 32, x);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&bars.f);
        if (!warp_wait(&bars.xf, ph, abort, err, 84)) break;
        tc_fence_after();
        ld_cols(tl + L::tK + tb, x);
#pragma unroll
        for (int j = 0; j < kTok; ++j) u[j] += x[j];
        float y[kTok];   // dV
        with_tokens(gates.bet, [&](int j, float g) { y[j] = g * u[j]; });
        with_tokens(gates.gam, [&](int j, float g) { x[j] = -g * y[j]; });
        put_pieces<PS, 0>(tl + L::tF + tb / 2, 32, x);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&bars.uw);
        const float glast = *gates.last;
        if (!STATE) {
#pragma unroll
          for (int j = 0; j < kTok; ++j) x[j] = u[j];
          put_pieces<PG, PG>(kNoTmem, 0, x, p.dup + at * kWF, lane, kChunk, tb);
          fetch_pieces<PS, kTok>(p.ep + at * kWF, lane, kChunk, tb, x);
#pragma unroll
          for (int j = 0; j < kTok; ++j) x[j] *= u[j];
          const float s = sum_columns(x);
          if ((lane & 1) == 0) p.edu[at * kChunk + tb + lane / 2] = s;
        }
        if (!STATE) {
          staged<T>(stage + L::kOffV, tb, lcol, x);
#pragma unroll
          for (int j = 0; j < kTok; ++j) x[j] *= y[j];
          const float s = sum_columns(x);
          if ((lane & 1) == 0) p.vdv[at * kChunk + tb + lane / 2] = s;
          // on to the chunk before: the tokens' sums, each in two lanes
          sds += warp_sum((lane & 1) == 0 ? p.odo[at * kChunk + tb + lane / 2] - s : 0.f);
          const int64_t tok = (int64_t)c * kChunk + tb;
          if (on)
            store_tokens(static_cast<T*>(p.dv_) + ((span.b * p.time + span.t0 + tok) * p.hv + h) * p.dv + col,
                         (int64_t)p.hv * p.dv, (int)min(span.n - tok, (int64_t)kTok), y);
        }
        fence_proxy_async();   // what this stage held is read before bulk copies may replace it
        if (!warp_wait(&bars.ds, ph, abort, err, 85)) break;
        tc_fence_after();
        {
          float d[HK];
          ld_cols(tl + L::tD + kb, d);
#pragma unroll
          for (int a = 0; a < HK; ++a) st[a] = glast * st[a] + d[a];
        }
        tc_fence_before();
        warp_arrive(&bars.empty[R::stage(i)]);
        if (i + 1 < nc) {
          warp_arrive(&bars.share[q]);   // the other quarters' columns are read before pieces go over them
          if (!warp_wait(&bars.share[q], ph, abort, err, 86)) break;
          tc_fence_after();
          put_state(c - 1);
        }
      }
      if (*abort) {
      } else if (STATE) {
        store_column(border(p.seg_ds, span.g), pitch, HK, st);
      } else if (span.first && p.ds_init != nullptr && on) {
        store_column(p.ds_init + sbase() + col, p.dv, p.dk - kb, st);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (STATE) wait_for_last();
}

template <int DKP, typename T, bool STATE>
cudaError_t run_rscan(const Params& p, cudaStream_t s) {
  constexpr int smem = RLayout<DKP, T>::kBytes;
  const double rows = (double)p.bound * kChunk * p.hv;
  int* err = device_error_flag();
  if (err == nullptr) return cudaErrorInvalidValue;
  LaunchTimer t(STATE ? "delta_rscan_state_kernel" : "delta_rscan_kernel", s, rows * 2.0 * p.dv * sizeof(T),
                rows * 6.0 * p.dk * p.dv);
  cudaError_t e = allow_smem<rscan_kernel<DKP, T, STATE>>(smem);
  if (e != cudaSuccess) return e;
  const unsigned spans = (unsigned)(p.seg > 0 ? p.nsegs : p.nseq);
  cudaLaunchAttribute beside{};
  beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  beside.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(spans * p.hv * ((p.dv + kLanes - 1) / kLanes));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &beside;
  cfg.numAttrs = STATE ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, rscan_kernel<DKP, T, STATE>, p, err);
}

template <typename T>
cudaError_t pick_rscan(const Params& p, bool state_only, cudaStream_t s) {
  if (state_only) return p.dk <= 64 ? run_rscan<64, T, true>(p, s) : run_rscan<128, T, true>(p, s);
  return p.dk <= 64 ? run_rscan<64, T, false>(p, s) : run_rscan<128, T, false>(p, s);
}

}  // namespace

cudaError_t launch_rscan(const Params& p, int dtype, bool state_only, cudaStream_t s) {
  if (dtype == 1) return pick_rscan<__nv_bfloat16>(p, state_only, s);
  if (dtype == 2) return pick_rscan<__half>(p, state_only, s);
  return pick_rscan<float>(p, state_only, s);
}

}  // namespace delta
}  // namespace qrb
