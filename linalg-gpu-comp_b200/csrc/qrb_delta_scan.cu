// The forward recurrence of the gated delta rule over the chunks of one sequence (mathematics in
// qrb_delta.cuh, data flow in qrb_delta_tc.cuh).
//
// The columns of the state evolve independently: a block owns one (sequence, value head, up to 128
// value columns) and walks its chunks.  Four threads share a column, each with a quarter of its state
// in fp32 registers for the whole sequence.  Per chunk, all transposed (lane = value column):
//     K S0 -> e0 = v - gamma (K S0), F = beta e0 -> X F -> e = e0 + X F, u = beta e, W = tail u
//     -> K^T W -> S = gamma_last S + K^T W -> pieces of S for the next chunk,
// a chain of three products with register work between them.  Q S0 and P u, which o is made of, run
// in the shadow of that work (the first is scaled in place and the second added to it), and o is stored
// in the shadow of the next chunk's K S0.  Sixteen warps, because the register work between two
// products is bound by latency; a thread beside them issues the MMAs (it is held up while the tensor
// cores' queue is full, which in a computing warp made every other one wait for it) and another loads
// the chunk tiles by bulk copies, two chunks in flight where they fit (issuing those takes 800 cycles a
// chunk).  An N = 64 MMA takes 47 cycles by itself, 60 to 120 while the warps use tensor memory.
// Measured (dk = dv = 128): 5.6 us a chunk in bf16, 24 packed sequences of 16384 tokens with 32 heads 332 us
// (58 chunks an SM); 7.8 us where it stores for a backward pass, which moves 240 KB a chunk.
#include "qrb_delta_tc.cuh"
#include "qrb_ring.cuh"

namespace qrb {
namespace delta {
namespace {

enum Mode { kOut, kStore, kState };   // of the forward recurrence, see scan_kernel

template <int DKP, typename T, int PS, int MODE>
struct ScanLayout {
  static constexpr int PX = kChainPieces;
  static constexpr int P = Pieces<T>::kIn;
  static constexpr int kK = tile_bytes(kChunk, P, DKP);
  static constexpr int kX = tile_bytes(kChunk, PX, kChunk), kP = tile_bytes(kChunk, PS, kChunk);
  static constexpr int kV = kChunk * kLanes * (int)sizeof(T);
  static constexpr int kGates = 3 * kChunk * 4;
  static constexpr int kOffX = kK, kOffV = kOffX + kX, kOffQ = kOffV + kV, kOffP = kOffQ + kK, kOffD = kOffP + kP;
  // a multiple of 1024; gates apart
  static constexpr int kStage = MODE == kState ? kOffQ : kOffD + (MODE == kStore ? kV : 0);
  static constexpr int kStages = 2 * (kStage + kGates) + 256 + 1024 <= kSmemLimit ? 2 : 1;
  static constexpr int kOffG = kStages * kStage;
  static constexpr int kBar = kOffG + kStages * kGates;
  static constexpr int kBytes = kBar + 256 + 1024;   // 1024: alignment
  static_assert(kBytes <= kSmemLimit, "shared memory of one block");
  // tensor memory columns: pieces of S, then K^T W over them (they are read by then; the warps that share
  // lanes meet before they are written again) | K S0, then X F | Q S0, then P u | F, then W | U
  static constexpr uint32_t kSp = PS * (DKP / 2);
  static constexpr uint32_t tS = 0, tD = 0, tK = kSp > (uint32_t)DKP ? kSp : DKP, tQ = tK + 64, tF = tQ + 64,
                            tU = tF + 32 * PX;
  static_assert(tU + 32 * PS <= 512, "tensor memory");
};

struct ScanBars {
  uint64_t full[2], empty[2], sp, ks, qs, f, xf, uw, sq, ds, pu, share[4], drain;   // full, empty: see qrb_ring.cuh
  uint32_t tmem;
  int abort;
  Span span;   // here, not in registers that the loops need
};
static_assert(sizeof(ScanBars) <= 256, "barrier block");

// kStore: for a backward pass, keep every chunk's first state, e and the sums o.do instead of o.
// kState: only the state, of every segment but a sequence's last: from the initial state for the first,
// else from zero; and one more block per head for the segment's transition, its columns those of the
// state that the identity and v = 0 become.
// CUT: sequences may be cut into segments.  Apart, since what a segment has to remember costs whole
// sequences registers and 6% (24 packed prompts, 32 heads: 326 against 348 us).
template <int DKP, typename T, int PS, int MODE, bool CUT>
__global__ void __launch_bounds__(kTcThreads, 1) scan_kernel(const __grid_constant__ Params p, int* err) {
  using L = ScanLayout<DKP, T, PS, MODE>;
  using R = Ring<L::kStages>;
  constexpr bool STORE = MODE == kStore, STATE = MODE == kState;
  constexpr int PG = Pieces<T>::kS;   // pieces of S0 kept for dq and dk
  constexpr int P = L::P, PX = L::PX, HK = DKP / kParts;   // HK: state rows of one thread
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                       ~uintptr_t(1023));
  ScanBars& bars = *reinterpret_cast<ScanBars*>(sm + L::kBar);
  volatile int* abort = &bars.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nb = (p.dv + kLanes - 1) / kLanes, nbx = nb + STATE;
  const int vb = blockIdx.x % nbx, sh = blockIdx.x / nbx, h = sh % p.hv;
  if (STATE) let_next_start();   // rscan's state-only pass, which needs nothing from this one
  const Span mine = span_at<CUT>(p, sh / p.hv);
  const bool unit = STATE && vb == nb;
  if (mine.nc < 0 || (STATE && (mine.last || (unit && mine.first)))) return;
  const int hk = h / p.group, nc = mine.nc, slot0 = mine.slot0;
  // 32-column groups that hold columns
  const int quarters = unit ? DKP / 32 : min(4, (p.dv - vb * kLanes + 31) / 32);

  if (tid == 0) {
    mbar_init(&bars.full[0], 1);
    mbar_init(&bars.full[1], 1);
    for (uint64_t* x : {&bars.ks, &bars.qs, &bars.xf, &bars.ds, &bars.pu, &bars.drain}) mbar_init(x, 1);
    for (uint64_t* x : {&bars.sp, &bars.f, &bars.uw, &bars.sq, &bars.empty[0], &bars.empty[1]})
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
    // ---------------- loads: one thread ----------------
    if (lane == 0) {
      int c = 0;
      for (; c < nc; ++c) {
        const int stage = R::stage(c);
        // the chunk that held this stage is done with: all its products and reads
        if (c >= L::kStages && !mbar_wait_abort(&bars.empty[stage], R::phase(c - L::kStages), abort, err, 51)) break;
        unsigned char* d = sm + stage * L::kStage;
        uint64_t* bar = &bars.full[stage];
        const size_t qk = ((size_t)(slot0 + c) * p.hk + hk) * L::kK, at = slot_head(p, slot0 + c, h);
        mbar_arrive_expect_tx(bar, L::kStage + L::kGates);
        bulk_load(d, p.kt + qk, L::kK, bar);
        bulk_load(sm + L::kOffG + stage * L::kGates, p.gates + at * 3 * kChunk, L::kGates, bar);
        bulk_load(d + L::kOffV, p.vt + (at * nb + (unit ? 0 : vb)) * L::kV, L::kV, bar);
        bulk_load(d + L::kOffX, p.xt + at * L::kX, L::kX, bar);
        if (STATE) continue;
        bulk_load(d + L::kOffQ, p.qt + qk, L::kK, bar);
        bulk_load(d + L::kOffP, p.pt + at * L::kP, L::kP, bar);
        if (STORE) bulk_load(d + L::kOffD, p.dot + (at * nb + vb) * L::kV, L::kV, bar);
      }
      if (*abort)   // loads in flight must land before the block's memory goes
        for (int s = 0; s < L::kStages; ++s)
          if (c > s) mbar_wait(&bars.full[s], R::phase(c - 1 - s), 1u << 22);
    }
  } else if (warp == kIssuer) {
    // ---------------- MMAs: one thread ----------------
    if (lane == 0) {
      for (int c = 0; c < nc; ++c) {
        const uint32_t ph = c & 1, sb = smem_u32(sm + R::stage(c) * L::kStage);
        if (!mbar_wait_abort(&bars.full[R::stage(c)], R::phase(c), abort, err, 52)) break;
        if (!mbar_wait_abort(&bars.sp, ph, abort, err, 53)) break;
        tc_fence_after();
        mma_pieces<64, DKP, false, PS, P, PS>(tmem + L::tK, tmem + L::tS, DKP / 2, sb, 0);
        mma_commit(&bars.ks);
        if (!mbar_wait_abort(&bars.f, ph, abort, err, 54)) break;
        tc_fence_after();
        mma_pieces<64, 64, false, PX, PX, PX>(tmem + L::tK, tmem + L::tF, 32, sb + L::kOffX, 0);
        mma_commit(&bars.xf);
        if (!STATE) {
          // the last chunk's o is read
          if (c > 0 && !mbar_wait_abort(&bars.empty[R::stage(c - 1)], R::phase(c - 1), abort, err, 55)) break;
          tc_fence_after();
          mma_pieces<64, DKP, false, PS, P, PS>(tmem + L::tQ, tmem + L::tS, DKP / 2, sb + L::kOffQ, 0);
          mma_commit(&bars.qs);
        }
        if (!mbar_wait_abort(&bars.uw, ph, abort, err, 56)) break;
        if (!STATE && !mbar_wait_abort(&bars.qs, ph, abort, err, 57)) break;   // the pieces of S are read
        tc_fence_after();
        mma_pieces<DKP, 64, true, PX, P, PX>(tmem + L::tD, tmem + L::tF, 32, sb, 0);
        mma_commit(&bars.ds);
        if (STATE) continue;
        if (!mbar_wait_abort(&bars.sq, ph, abort, err, 58)) break;
        tc_fence_after();
        mma_pieces<64, 64, false, PS, PS, PS>(tmem + L::tQ, tmem + L::tU, 32, sb + L::kOffP, 1);
        mma_commit(&bars.pu);
      }
      if (*abort) {   // MMAs in flight must end before tensor memory goes
        mma_commit(&bars.drain);
        mbar_wait(&bars.drain, 0, 1u << 22);
      }
    }
  } else {
    const Span& span = CUT ? bars.span : mine;
    const bool first = !CUT || span.first, last = !CUT || span.last;
    const int q = warp & 3, part = warp >> 2;
    if (q < quarters) {   // warps without columns have nothing to add
      const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
      const int lcol = 32 * q + lane, col = vb * kLanes + lcol;  // value column in the block, in the head
      const int tile = vb * 4 + q;                              // its 32-column tile
      const int tb = kTok * part, kb = HK * part;               // first token, first state row
      const bool on = col < p.dv;
      auto sbase = [&] { return (((size_t)span.seq * p.hv + h) * p.dk + kb) * p.dv; };
      // S at the borders of segments: dense rows of all lanes, DKP of them
      const int pitch = nb * kLanes;
      auto border = [&](int g) { return p.seg_s + (((size_t)g * p.hv + h) * DKP + kb) * pitch + col; };
      constexpr int kWS = tile_bytes(kTile, PS, DKP), kWF = tile_bytes(kTile, PS, kChunk);
      float st[HK];
      if (unit) {
#pragma unroll
        for (int j = 0; j < HK; ++j) st[j] = kb + j == lcol ? 1.f : 0.f;
      } else if (!STATE && !(first && last)) {
        load_column(border(span.g), pitch, HK, true, st);
      } else if (first && p.s_init != nullptr) {
        load_column(p.s_init + sbase() + min(col, p.dv - 1), p.dv, p.dk - kb, on, st);
      } else {
#pragma unroll
        for (int j = 0; j < HK; ++j) st[j] = 0.f;
      }
      if (STATE && first) store_column(border(span.g), pitch, HK, st);
      auto put_state = [&](int c) {
        float y[HK];
#pragma unroll
        for (int i = 0; i < HK; ++i) y[i] = st[i];
        unsigned char* to = STORE ? p.s0p + (slot_head(p, slot0 + c, h) * p.nv + tile) * kWS : nullptr;
        // all pieces where the backward recurrence takes <S', dS'> from them, else those dq and dk need
        if (STORE && (nc - c) % kAnchor == 0) put_pieces<PS, PS>(tl + L::tS + kb / 2, DKP / 2, y, to, lane, DKP, kb);
        else put_pieces<PS, STORE ? PG : 0>(tl + L::tS + kb / 2, DKP / 2, y, to, lane, DKP, kb);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&bars.sp);
      };
      if (nc > 0) put_state(0);
      for (int c = 0; c < nc; ++c) {
        const uint32_t ph = c & 1;
        const unsigned char* stage = sm + R::stage(c) * L::kStage;
        const Gates gates(sm + L::kOffG + R::stage(c) * L::kGates, tb);
        float e[kTok], x[kTok];
        if (!warp_wait(&bars.full[R::stage(c)], R::phase(c), abort, err, 61)) break;
        staged<T>(stage + L::kOffV, tb, lcol, e);
        if (unit) {
#pragma unroll
          for (int i = 0; i < kTok; ++i) e[i] = 0.f;
        }
        if (!warp_wait(&bars.ks, ph, abort, err, 62)) break;
        tc_fence_after();
        ld_cols(tl + L::tK + tb, x);
        with_tokens(gates.gam, [&](int i, float g) { e[i] -= g * x[i]; });
        with_tokens(gates.bet, [&](int i, float g) { x[i] = g * e[i]; });
        put_pieces<PX, 0>(tl + L::tF + tb / 2, 32, x);
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&bars.f);
        if (!warp_wait(&bars.xf, ph, abort, err, 64)) break;
        tc_fence_after();
        ld_cols(tl + L::tK + tb, x);
#pragma unroll
        for (int i = 0; i < kTok; ++i) x[i] += e[i];   // x: e
        with_tokens(gates.bet, [&](int i, float g) { e[i] = g * x[i]; });   // e: u
        {
          float y[kTok];
          with_tokens(gates.tail, [&](int i, float g) { y[i] = g * e[i]; });
          if (!STATE) put_pieces<PS, 0>(tl + L::tU + tb / 2, 32, e);
          put_pieces<PX, 0>(tl + L::tF + tb / 2, 32, y);
        }
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&bars.uw);
        if (STORE)
          put_pieces<PS, PS>(kNoTmem, 0, x, p.ep + (slot_head(p, slot0 + c, h) * p.nv + tile) * kWF, lane, kChunk, tb);
        if (!STATE) {
          if (!warp_wait(&bars.qs, ph, abort, err, 63)) break;
          tc_fence_after();
          ld_cols(tl + L::tQ + tb, x);   // scale gamma Q S0 goes back, P u is added to it there
          {
            uint32_t y[kTok];
            with_tokens(gates.gam, [&](int i, float g) { y[i] = __float_as_uint(p.scale * g * x[i]); });
            st_cols(tl + L::tQ + tb, y);
          }
          tmem_st_wait();
          tc_fence_before();
          warp_arrive(&bars.sq);
        }
        const float glast = *gates.last;
        if (!warp_wait(&bars.ds, ph, abort, err, 65)) break;
        tc_fence_after();
        {
          float y[HK];
          ld_cols(tl + L::tD + kb, y);
#pragma unroll
          for (int i = 0; i < HK; ++i) st[i] = glast * st[i] + y[i];
        }
        if (c + 1 < nc) {
          tc_fence_before();
          warp_arrive(&bars.share[q]);   // the other quarters' columns of K^T W are read too
          if (!warp_wait(&bars.share[q], ph, abort, err, 66)) break;
          tc_fence_after();
          put_state(c + 1);
        }
        if (!STATE) {
          if (!warp_wait(&bars.pu, ph, abort, err, 67)) break;
          tc_fence_after();
          ld_cols(tl + L::tQ + tb, x);
        }
        if (STORE) staged<T>(stage + L::kOffD, tb, lcol, e);
        tc_fence_before();
        fence_proxy_async();   // what this stage held is read before bulk copies may replace it
        warp_arrive(&bars.empty[R::stage(c)]);
        if (STORE) {
#pragma unroll
          for (int i = 0; i < kTok; ++i) x[i] *= e[i];
          const float s = sum_columns(x);
          if ((lane & 1) == 0) p.odo[(slot_head(p, slot0 + c, h) * p.nv + tile) * kChunk + tb + lane / 2] = s;
        } else if (MODE == kOut && on) {
          const int64_t tok = (int64_t)c * kChunk + tb;
          store_tokens(static_cast<T*>(p.o) + span.b * p.os.b + (span.t0 + tok) * p.os.t + h * p.os.h + col, p.os.t,
                       (int)min(span.n - tok, (int64_t)kTok), x);
        }
      }
      if (*abort) {
      } else if (unit) {
        store_column(p.seg_a + (((size_t)span.g * p.hv + h) * DKP + kb) * DKP + lcol, DKP, HK, st);
      } else if (STATE) {
        store_column(border(span.g + 1), pitch, HK, st);
      } else if (last && p.s_end != nullptr && on) {
        store_column(p.s_end + sbase() + col, p.dv, p.dk - kb, st);
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

template <int DKP, typename T, int PS, int MODE, bool CUT>
cudaError_t run_cut(const Params& p, cudaStream_t s) {
  constexpr int smem = ScanLayout<DKP, T, PS, MODE>::kBytes;
  const unsigned spans = (unsigned)(CUT ? p.nsegs : p.nseq);
  const unsigned grid = spans * p.hv * ((p.dv + kLanes - 1) / kLanes + (MODE == kState));
  const double rows = (double)p.bound * kChunk * p.hv;
  int* err = device_error_flag();
  if (err == nullptr) return cudaErrorInvalidValue;
  const char* name = MODE == kStore ? "delta_scan_store_kernel" : MODE == kState ? "delta_scan_state_kernel" : "delta_scan_kernel";
  LaunchTimer t(name, s, rows * 2.0 * p.dv * sizeof(T), rows * 6.0 * p.dk * p.dv);
  cudaError_t e = allow_smem<scan_kernel<DKP, T, PS, MODE, CUT>>(smem);
  if (e != cudaSuccess) return e;
  scan_kernel<DKP, T, PS, MODE, CUT><<<grid, kTcThreads, smem, s>>>(p, err);
  return cudaGetLastError();
}

template <int DKP, typename T, int PS, int MODE>
cudaError_t run_scan(const Params& p, cudaStream_t s) {
  if constexpr (MODE == kState) return run_cut<DKP, T, PS, MODE, true>(p, s);
  else return p.seg > 0 ? run_cut<DKP, T, PS, MODE, true>(p, s) : run_cut<DKP, T, PS, MODE, false>(p, s);
}

template <typename T>
cudaError_t pick_scan(const Params& p, bool state_only, cudaStream_t s) {
  constexpr int B = kBackPieces, S = Pieces<T>::kS;
  if (state_only) return p.dk <= 64 ? run_scan<64, T, B, kState>(p, s) : run_scan<128, T, B, kState>(p, s);
  if (p.backward) return p.dk <= 64 ? run_scan<64, T, B, kStore>(p, s) : run_scan<128, T, B, kStore>(p, s);
  return p.dk <= 64 ? run_scan<64, T, S, kOut>(p, s) : run_scan<128, T, S, kOut>(p, s);
}

}  // namespace

cudaError_t launch_scan(const Params& p, int dtype, bool state_only, cudaStream_t s) {
  if (dtype == 1) return pick_scan<__nv_bfloat16>(p, state_only, s);
  if (dtype == 2) return pick_scan<__half>(p, state_only, s);
  return pick_scan<float>(p, state_only, s);
}

}  // namespace delta
}  // namespace qrb
