// C ABI of the gated delta rule (include/qrb200_nn.h): argument checks, workspace layout and
// the launch sequence.
//   forward:  [plan] prep, scan
//   backward: [plan] prep, scan (keeping every chunk's state and e), rscan, grad
// where long sequences are cut into segments: prep, [state-only scan, state-only rscan], join, scan, ...
// Backward repeats the forward recurrence instead of asking the caller to keep 4 dk dv bytes per
// 64 tokens and head between the passes.
#include <cstdarg>
#include <cstdio>

#include "../../include/qrb200_nn.h"
#include "qrb_delta.cuh"

namespace {

using qrb::delta::kChunk;
using qrb::delta::kTile;
using qrb::delta::Params;

int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return qrb::set_error(status, buf);
}

#define TRY(x)                   \
  do {                           \
    int _s = (x);                \
    if (_s != QRB_OK) return _s; \
  } while (0)
#define CUDA(x, what)                                                                                 \
  do {                                                                                                \
    cudaError_t _e = (x);                                                                             \
    if (_e != cudaSuccess)                                                                            \
      return fail(QRB_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(_e), cudaGetErrorString(_e));   \
  } while (0)

size_t al(size_t x) { return (x + 255) & ~size_t(255); }

int pieces_in(int dtype) { return dtype == QRB_BF16 ? 1 : (dtype == QRB_F16 ? 2 : 3); }
int pieces_s(int dtype) { return dtype == QRB_F32 ? 3 : 2; }

int check_sizes(int dtype, int hk, int hv, int dk, int dv) {
  if (dtype != QRB_F32 && dtype != QRB_BF16 && dtype != QRB_F16)
    return fail(QRB_ERR_INVALID_ARG, "dtype must be QRB_F32, QRB_BF16 or QRB_F16 (got %d)", dtype);
  if (hk < 1 || hv < 1 || hv % hk != 0)
    return fail(QRB_ERR_INVALID_ARG, "hv must be a positive multiple of hk (got hk = %d, hv = %d)", hk, hv);
  if (dk < 1 || dv < 1) return fail(QRB_ERR_INVALID_ARG, "dk and dv must be >= 1 (got %d, %d)", dk, dv);
  if (dk > QRB_DELTA_MAX_DK || dv > QRB_DELTA_MAX_DV)
    return fail(QRB_ERR_UNSUPPORTED, "dk = %d, dv = %d exceed %d, %d", dk, dv, QRB_DELTA_MAX_DK, QRB_DELTA_MAX_DV);
  if (hv > 65535) return fail(QRB_ERR_UNSUPPORTED, "hv = %d exceeds 65535", hv);
  return QRB_OK;
}

int check_ptr(const void* p, const char* name, size_t align) {
  if (p == nullptr) return fail(QRB_ERR_INVALID_ARG, "%s is null", name);
  if ((reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0)
    return fail(QRB_ERR_INVALID_ARG, "%s must be %zu-byte aligned", name, align);
  return QRB_OK;
}

// Chunk slots: packed sequences each round up once, and the rows behind the last one take the rest.
int64_t chunk_slots(const qrb_delta_args& a) {
  if (a.seq_offsets == nullptr) return a.nseq * ((a.time + kChunk - 1) / kChunk);
  return (a.time + (int64_t)(kChunk - 1) * (a.nseq + 1)) / kChunk;
}

int check_args(const qrb_delta_args* a) {
  if (a == nullptr) return fail(QRB_ERR_INVALID_ARG, "args is null");
  TRY(check_sizes(a->dtype, a->hk, a->hv, a->dk, a->dv));
  if (a->batch < 0 || a->time < 0 || a->nseq < 0)
    return fail(QRB_ERR_INVALID_ARG, "batch, time and nseq must be >= 0 (got %lld, %lld, %lld)", (long long)a->batch,
                (long long)a->time, (long long)a->nseq);
  if (a->seq_offsets == nullptr && a->nseq != a->batch)
    return fail(QRB_ERR_INVALID_ARG, "without seq_offsets nseq must be batch");
  if (a->seq_offsets != nullptr && a->batch != 1)
    return fail(QRB_ERR_INVALID_ARG, "packed sequences need batch == 1 (got %lld)", (long long)a->batch);
  const int64_t nv = (a->dv + kTile - 1) / kTile;
  if (a->time > INT32_MAX || a->nseq > INT32_MAX / 2 || a->nseq * a->hv * nv > INT32_MAX || chunk_slots(*a) > INT32_MAX)
    return fail(QRB_ERR_UNSUPPORTED, "too many sequences or tokens (nseq = %lld, time = %lld)", (long long)a->nseq,
                (long long)a->time);
  return QRB_OK;
}

// Segments of `seg` chunks (0: whole sequences) and how many there may be at most.  With one chunk of the
// full recurrence as the unit (5.6 us at dk = dv = 128 in bf16), one of the state-only pass takes about
// as much (0.6 in fp32), a join's step 1/4 and the two launches 3.5: a sequence of nc chunks costs
// 2 seg + ns / 4 + 3.5 in ns segments, which is least at seg = sqrt(nc / 8) where there are SMs for so
// many.  One sequence, 16 heads of 128 x 128, bf16, as called: 512 tokens 63 us whole, 67 in four (captured
// 60 and 59); 1024 tokens 105 and 88; 4096 tokens 379 and 245; backward, whose chunks take longer, 512 tokens
// 189 us whole, 139 in four, 4096 tokens 1204 and 552.  The state-only pass has one more block per head, for
// the transition.
// Packed lengths are not known on the host: segments are cut as if one sequence held most of the tokens,
// which costs little where it does not (a sequence of one segment has no first pass), unless the
// sequences alone nearly fill the card.  7 packed sequences, 6 heads of 64 x 64, 3001 tokens, fp16, backward:
// 610 us whole, 181 cut.
struct Segments {
  int seg, nsegs;
};
Segments segments(const qrb_delta_args& a, bool backward) {
  const int64_t nb = (a.dv + 127) / 128;
  const int64_t room = qrb::sm_count() / (a.hv * (nb + 1));   // segments with an SM for each of their blocks
  const bool packed = a.seq_offsets != nullptr;
  Segments s{0, 0};
  // Two segments need no transition, so they may have room where more have not; then the first pass is
  // half a sequence's, which pays where it is clearly cheaper than the second: 4 x 2048 tokens, 16 heads
  // of 128 x 128, backward in bf16 792 us whole, 673 in halves, forward in fp32 615 and 568, but in bf16 258
  // and 279.  (Where there is room for exactly two with their transition, `room` = 2 nseq, the test of cost at
  // the end is never met, so 25 to 37 heads and sequences run whole at any length: forward in bf16 that is
  // right, 8192 tokens of 32 heads 809 us whole and 832 in halves, backward it is not, 2564 and 1901.)
  const bool halves = !packed && room < 2 * a.nseq && (backward || a.dtype == QRB_F32) &&
                      qrb::sm_count() / (a.hv * nb) >= 2 * a.nseq;
  if (a.nseq < 1 || (packed ? 2 * room < 3 * a.nseq : room < 2 * a.nseq && !halves)) return s;
  const int64_t nc = packed ? chunk_slots(a) : (a.time + kChunk - 1) / kChunk;
  const int64_t each = packed ? room : halves ? 2 : room / a.nseq;
  if (nc < (packed || halves ? 16 : 6)) return s;
  int64_t seg = (nc + each - 1) / each;
  while (8 * seg * seg < nc && !halves) ++seg;
  if (packed) {
    if (seg < 3) seg = 3;
    s.nsegs = (int)(nc / seg + a.nseq);
  } else {
    const int64_t ns = (nc + seg - 1) / seg;
    if (!halves && 8 * seg + ns + (backward ? 6 : 14) > 4 * nc) return s;
    s.nsegs = (int)(ns * a.nseq);
  }
  s.seg = (int)seg;
  return s;
}

struct Layout {
  size_t cstart, kt, qt, xt, pt, gates, gsum, s0p, dsp, ep, dup, odo, vdv, edu, sds, s_last, vt, dot, dop, total;
  size_t seg_s, seg_a, seg_ds;
};

Layout layout(const qrb_delta_args& a, bool backward) {
  using namespace qrb::delta;
  const size_t n = (size_t)chunk_slots(a), dkp = a.dk <= 64 ? 64 : 128, nv = (a.dv + kTile - 1) / kTile;
  const int pi = pieces_in(a.dtype), ps = backward ? kBackPieces : pieces_s(a.dtype);
  Layout l{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += al(bytes);
    return o;
  };
  l.cstart = take(a.seq_offsets != nullptr ? (3 * a.nseq + 2) * 4 : 0);
  l.kt = take(n * a.hk * tile_bytes(kChunk, pi, dkp));
  l.qt = take(n * a.hk * tile_bytes(kChunk, pi, dkp));
  l.xt = take(n * a.hv * tile_bytes(kChunk, kChainPieces, kChunk));
  l.pt = take(n * a.hv * tile_bytes(kChunk, ps, kChunk));
  l.gates = take(n * a.hv * 3 * kChunk * 4);
  const size_t staged = n * a.hv * ((a.dv + 127) / 128) * kChunk * 128 * (a.dtype == QRB_F32 ? 4 : 2);
  l.vt = take(staged);
  const Segments g = segments(a, backward);
  const size_t cells = (size_t)g.nsegs * a.hv * dkp * 4;   // of one column of every border
  l.seg_s = take(cells * ((a.dv + 127) / 128) * 128);
  l.seg_a = take(cells * dkp);
  if (backward) l.seg_ds = take(cells * ((a.dv + 127) / 128) * 128);
  if (backward) {
    l.dot = take(staged);
    if (grad_on_tc(a.dtype)) l.dop = take(n * a.hv * nv * tile_bytes(kTile, pi, kChunk));
    l.gsum = take(n * a.hv * kChunk * 8);
    l.s0p = take(n * a.hv * nv * tile_bytes(kTile, ps, dkp));
    l.dsp = take(n * a.hv * nv * tile_bytes(kTile, ps, dkp));
    l.ep = take(n * a.hv * nv * tile_bytes(kTile, ps, kChunk));
    l.dup = take(n * a.hv * nv * tile_bytes(kTile, ps, kChunk));
    l.odo = take(n * a.hv * nv * kChunk * 4);
    l.vdv = take(n * a.hv * nv * kChunk * 4);
    l.edu = take(n * a.hv * nv * kChunk * 4);
    l.sds = take(n * a.hv * nv * 4 * 4);
    l.s_last = take((size_t)a.nseq * a.hv * a.dk * a.dv * 4);
  }
  l.total = at;
  return l;
}

int check_device() {
  int dev = 0, major = 0;
  CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  static int cache[64] = {0};
  if (dev < 64) major = cache[dev];
  if (major == 0) {
    CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev), "cudaDeviceGetAttribute");
    if (dev < 64) cache[dev] = major;
  }
  if (major != 10)
    return fail(QRB_ERR_DEVICE, "device %d has compute capability %d.x; libqrb200 needs sm_100", dev, major);
  return QRB_OK;
}

qrb::delta::Strides st(const qrb_strides& s) { return {s.batch, s.time, s.head}; }

int run(const qrb_delta_args* a, void* ws, size_t wsb, void* stream, bool backward) {
  TRY(check_args(a));
  if (a->nseq == 0) {
    if (a->seq_offsets == nullptr || a->time == 0 || !a->zero_tail) return QRB_OK;
    return fail(QRB_ERR_INVALID_ARG, "seq_offsets must hold at least one sequence");
  }
  const size_t es = a->dtype == QRB_F32 ? 4 : 2;
  if (a->time > 0) {
    TRY(check_ptr(a->q, "q", es));
    TRY(check_ptr(a->k, "k", es));
    TRY(check_ptr(a->v, "v", es));
    TRY(check_ptr(a->g, "g", 4));
    TRY(check_ptr(a->beta, "beta", 4));
    if (!backward) {
      TRY(check_ptr(a->o, "o", es));
    } else {
      TRY(check_ptr(a->d_o, "d_o", es));
      TRY(check_ptr(a->dq, "dq", es));
      TRY(check_ptr(a->dk_, "dk", es));
      TRY(check_ptr(a->dv_, "dv", es));
      TRY(check_ptr(a->dg, "dg", 4));
      TRY(check_ptr(a->dbeta, "dbeta", 4));
    }
  }
  const Layout l = layout(*a, backward);
  if (l.total > 0) {
    if (ws == nullptr || wsb < l.total)
      return fail(QRB_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given%s", l.total, wsb,
                  ws == nullptr ? " (null)" : "");
    if ((reinterpret_cast<uintptr_t>(ws) & 255u) != 0)
      return fail(QRB_ERR_INVALID_ARG, "workspace must be 256-byte aligned");
  }
  TRY(check_device());
  unsigned char* w = static_cast<unsigned char*>(ws);
  Params p{};
  p.hk = a->hk;
  p.hv = a->hv;
  p.group = a->hv / a->hk;
  p.dk = a->dk;
  p.dv = a->dv;
  p.nv = (a->dv + kTile - 1) / kTile;
  p.nseq = (int)a->nseq;
  p.nchunk = a->seq_offsets != nullptr ? 0 : (int)((a->time + kChunk - 1) / kChunk);
  p.bound = (int)chunk_slots(*a);
  p.time = a->time;
  p.offsets = a->seq_offsets;
  p.cstart = reinterpret_cast<int32_t*>(w + l.cstart);
  p.order = p.cstart + a->nseq + 1;
  p.segstart = p.order + a->nseq;
  const Segments g = segments(*a, backward);
  p.seg = g.seg;
  p.nsegs = g.nsegs;
  p.seg_s = reinterpret_cast<float*>(w + l.seg_s);
  p.seg_a = reinterpret_cast<float*>(w + l.seg_a);
  p.seg_ds = reinterpret_cast<float*>(w + l.seg_ds);
  p.scale = a->scale;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.d_o = a->d_o;
  p.g = a->g;
  p.beta = a->beta;
  p.qs = st(a->q_strides);
  p.ks = st(a->k_strides);
  p.vs = st(a->v_strides);
  p.gs = st(a->g_strides);
  p.bs = st(a->beta_strides);
  p.os = st(a->o_strides);
  p.dos = st(a->do_strides);
  p.s_init = a->initial_state;
  p.ds_end = a->dfinal_state;
  p.s_last = reinterpret_cast<float*>(w + l.s_last);
  p.s_end = backward ? p.s_last : a->final_state;
  p.ds_init = a->dinitial_state;
  p.o = a->o;
  p.dq = a->dq;
  p.dk_ = a->dk_;
  p.dv_ = a->dv_;
  p.dg = a->dg;
  p.dbeta = a->dbeta;
  p.zero_tail = a->seq_offsets != nullptr && a->zero_tail;
  p.backward = backward;
  p.kt = w + l.kt;
  p.qt = w + l.qt;
  p.xt = w + l.xt;
  p.pt = w + l.pt;
  p.vt = w + l.vt;
  p.dot = w + l.dot;
  p.dop = w + l.dop;
  p.gates = reinterpret_cast<float*>(w + l.gates);
  p.gsum = reinterpret_cast<double*>(w + l.gsum);
  p.s0p = w + l.s0p;
  p.dsp = w + l.dsp;
  p.ep = w + l.ep;
  p.dup = w + l.dup;
  p.odo = reinterpret_cast<float*>(w + l.odo);
  p.vdv = reinterpret_cast<float*>(w + l.vdv);
  p.edu = reinterpret_cast<float*>(w + l.edu);
  p.sds = reinterpret_cast<float*>(w + l.sds);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.offsets != nullptr) CUDA(qrb::delta::launch_plan(p, s), "delta plan launch");
  if (p.bound > 0) CUDA(qrb::delta::launch_prep(p, a->dtype, s), "delta chunk factor launch");
  if (p.seg > 0) {
    CUDA(qrb::delta::launch_scan(p, a->dtype, true, s), "delta segment launch");
    if (backward) CUDA(qrb::delta::launch_rscan(p, a->dtype, true, s), "delta backward segment launch");
    CUDA(qrb::delta::launch_join(p, s), "delta join launch");
  }
  CUDA(qrb::delta::launch_scan(p, a->dtype, false, s), "delta recurrence launch");
  if (backward) {
    CUDA(qrb::delta::launch_rscan(p, a->dtype, false, s), "delta backward recurrence launch");
    if (p.bound > 0) CUDA(qrb::delta::launch_grad(p, a->dtype, s), "delta gradient launch");
  }
  return QRB_OK;
}

}  // namespace

extern "C" {

size_t qrb_delta_workspace_size(const qrb_delta_args* a, int backward) {
  if (check_args(a) != QRB_OK) return 0;
  return layout(*a, backward != 0).total;
}

int qrb_delta_forward(const qrb_delta_args* a, void* ws, size_t wsb, void* stream) {
  return run(a, ws, wsb, stream, false);
}

int qrb_delta_backward(const qrb_delta_args* a, void* ws, size_t wsb, void* stream) {
  return run(a, ws, wsb, stream, true);
}

int qrb_delta_step(const qrb_delta_step_args* a, void* stream) {
  if (a == nullptr) return fail(QRB_ERR_INVALID_ARG, "args is null");
  TRY(check_sizes(a->dtype, a->hk, a->hv, a->dk, a->dv));
  if (a->batch < 0 || a->num_slots < 0)
    return fail(QRB_ERR_INVALID_ARG, "batch and num_slots must be >= 0 (got %lld, %lld)", (long long)a->batch,
                (long long)a->num_slots);
  if (a->batch > INT32_MAX / (a->hv * 8) || a->num_slots > INT32_MAX)
    return fail(QRB_ERR_UNSUPPORTED, "batch = %lld or num_slots = %lld is too large", (long long)a->batch,
                (long long)a->num_slots);
  if (a->slots == nullptr && a->batch > a->num_slots)
    return fail(QRB_ERR_INVALID_ARG, "batch = %lld rows need as many states (got %lld)", (long long)a->batch,
                (long long)a->num_slots);
  if (a->batch == 0) return QRB_OK;
  const size_t es = a->dtype == QRB_F32 ? 4 : 2;
  TRY(check_ptr(a->q, "q", es));
  TRY(check_ptr(a->k, "k", es));
  TRY(check_ptr(a->v, "v", es));
  TRY(check_ptr(a->g, "g", 4));
  TRY(check_ptr(a->beta, "beta", 4));
  TRY(check_ptr(a->o, "o", es));
  if (a->num_slots > 0) {
    TRY(check_ptr(a->state, "state", 4));
    TRY(check_ptr(a->state_out, "state_out", 4));
  }
  TRY(check_device());
  CUDA(qrb::delta::launch_step(*a, static_cast<cudaStream_t>(stream)), "delta step launch");
  return QRB_OK;
}

}  // extern "C"
