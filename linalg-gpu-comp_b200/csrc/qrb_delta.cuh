// Shared parts of the gated delta rule kernels (qrb_delta_*.cu).
//
// Per head the operator carries a state S (dk x dv) through a product of scaled
// Householder-like transforms,
//     S~_t = exp(g_t) S_{t-1},  u_t = beta_t (v_t - S~_t^T k_t),  S_t = S~_t + k_t u_t^T,
//     o_t = scale S_t^T q_t.
// Over a chunk of kChunk tokens the product has a compact-WY form, as the reflectors of a QR
// panel have.  With G the running sum of g in the chunk, D_ij = exp(G_i - G_j) (j <= i),
// gamma_i = exp(G_i), tail_i = exp(G_last - G_i), S0 / S' the states before / after it:
//     M_ij = D_ij k_i.k_j (j < i),   X = -M - M diag(beta) X   (strictly lower triangular),
//     E0 = V - diag(gamma) K S0,     e = E0 + X (beta E0),     u = beta e,
//     O  = scale diag(gamma) Q S0 + P u,   P_ij = scale D_ij q_i.k_j (j <= i),
//     S' = gamma_last S0 + K^T (tail u).
// X takes no division, so beta may be zero.  Backward, from dO and dS':
//     du = du0 + X^T (beta du0),  du0 = P^T dO + tail K dS',  dV = beta du,
//     dS0 = gamma_last dS' + scale (gamma Q)^T dO - (gamma K)^T dV,
//     Z_ij = scale D_ij dO_i.u_j (j <= i),  N_ij = -D_ij dV_i.u_j (j < i),
//     dQ = scale gamma dO S0^T + Z K,
//     dK = -gamma dV S0^T + tail u dS'^T + Z^T Q + (N + N^T) K,
//     dbeta_i = e_i.du_i,
//     dg_t = sum_{s >= t in the chunk} (o_s.do_s - v_s.dv_s) + <S', dS'>:
// scaling the state before token t by exp(x) is what g_t + x does, and v_s and o_s are the only
// ways in and out of the state after it.
//
// Precision: states, accumulators and gates are fp32 (G fp64).  Products run on the tensor cores
// with every fp32 operand split into bf16 pieces, x = x0 + x1 (+ x2): two pieces keep 2^-18 of x,
// three 2^-27; bf16 inputs are one piece and exact, fp16 inputs two and exact.  Products of pieces
// i, j with i + j below the piece count are added.  X, F = beta e0 and W = tail u, whose
// errors the state keeps, take three pieces; S0, P and u, which enter e and o once, two for the 16-bit
// types (with two everywhere the fp32 final state was 3e-6 off, so it is below 1e-6).  fp32 and the
// backward recurrences take three throughout: dg is the small difference of the sums above, and with two
// it was 2e-5 off, four to eight times the error of its terms.  dq and dk, rounded to their type in the
// end, take two pieces of the 16-bit types.
//
// Operand tiles are bf16 in blocks of 64 columns (128 bytes a row), the 16-byte units of a row
// XORed with row % 8, both in shared memory (where ldmatrix then reads without bank conflicts)
// and in the workspace (so that a tile moves with plain 16-byte copies).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/qrb200_nn.h"
#include "qrb_internal.cuh"

namespace qrb {
namespace delta {

constexpr int kChunk = 64;   // tokens per chunk
constexpr int kTile = 32;    // value columns per tile the recurrences leave for the gradient kernel
constexpr int kLanes = 128;  // value columns per block of the recurrences
constexpr float kMinLog = -120.f;   // exp(kMinLog) is 0 in fp32: a smaller g (-inf too) is the same decay

struct Strides {
  int64_t b, t, h;   // elements: batch, time, head (the last dimension is dense)
};

// One call, as the kernels see it.
struct Params {
  int hk, hv, group, dk, dv, nv;   // group = hv / hk, nv = value tiles
  int nseq, nchunk;                // nchunk: chunks a sequence of the dense layout has (0: packed)
  int bound;                       // chunk slots in the workspace
  int64_t time;
  const int32_t* offsets;          // packed layout: nseq + 1 token offsets
  int32_t* cstart;                 // packed layout: first chunk slot of each sequence
  int32_t* order;                  // packed layout: the sequences, longest first
  // Long sequences on few heads: segments of `seg` chunks run side by side (0: whole sequences; see
  // qrb_delta_join.cu).  segstart: packed layout, first segment of each sequence; nsegs: an upper bound.
  int seg, nsegs;
  int32_t* segstart;
  // [segment][hv]: S before it (dkp x nb*128), its transition (dkp x dkp), dS before it (for a first
  // segment: dS behind the sequence, which like S before it is copied since the caller's may be written over)
  float *seg_s, *seg_a, *seg_ds;
  float scale;
  const void *q, *k, *v, *d_o;
  const float *g, *beta;
  Strides qs, ks, vs, gs, bs, os, dos;
  const float *s_init, *ds_end;
  float *s_end, *ds_init;
  void *o, *dq, *dk_, *dv_;        // gradients are dense (batch, time, heads, d)
  float *dg, *dbeta;               // dense (batch, time, heads)
  int zero_tail, backward;         // zero the rows behind the last sequence
  // workspace, per chunk slot and head
  unsigned char *kt, *qt, *xt, *pt, *s0p, *dsp, *ep, *dup;
  unsigned char* dop;              // pieces of dO as tiles like du's, where grad_on_tc
  unsigned char *vt, *dot;         // v, dO: kChunk x 128 tiles, zero behind the sequence and dv
  float* gates;                    // gamma[64], tail[64], beta[64]
  double* gsum;                    // G[64]
  // backward, per chunk slot, head and tile: o.do, v.dv and e.du of 64 tokens, <S', dS'> in four parts
  float *odo, *vdv, *edu, *sds;
  float* s_last;                   // backward: every sequence's final state
};

template <typename T>
struct Pieces;   // kIn: pieces of an input, kS: of S0, P and u in the forward pass, and in dq, dk
template <>
struct Pieces<__nv_bfloat16> {
  static constexpr int kIn = 1, kS = 2;
};
template <>
struct Pieces<__half> {
  static constexpr int kIn = 2, kS = 2;
};
template <>
struct Pieces<float> {
  static constexpr int kIn = 3, kS = 3;
};
constexpr int kBackPieces = 3;   // of the backward recurrences
constexpr int kChainPieces = 3;  // of X, F and W
// (One bf16 piece of S0, P and u in o was tried for bf16 calls: its two products cancel in part, and o was
// 3.6e-3 off in place of 1.7e-3.)
// Backward: every kAnchor-th chunk from a sequence's end takes <S', dS'> from the states themselves, the
// others from the next chunk's by the same identity as dg within a chunk (see qrb_delta_rscan.cu).  The
// states' third pieces are then kept and read half as often; at every eighth dg was 1.8e-6 off.
constexpr int kAnchor = 2;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// Bytes per row of a tile with `pieces` pieces of `cols` columns each.
__host__ __device__ constexpr int row_blocks(int pieces, int cols) { return (pieces * cols + 63) / 64; }
__host__ __device__ constexpr int tile_bytes(int rows, int pieces, int cols) {
  return rows * 128 * row_blocks(pieces, cols);
}

// Byte offset of (row, col) in a tile of `rows` rows.
__device__ __forceinline__ uint32_t tile_off(int rows, int row, int col) {
  return (uint32_t)((col >> 6) * rows * 128 + row * 128 + ((((col >> 3) ^ row) & 7) << 4) + ((col & 7) << 1));
}

// The same for the tiles the recurrences leave behind (32 value columns as rows): 16-byte units of a
// row lie one tile column apart, so that a warp whose lanes own the rows writes 512 contiguous bytes,
// and ldmatrix still reads eight rows of a unit as 128 contiguous ones.
__device__ __forceinline__ uint32_t unit_off(int rows, int row, int col) {
  return (uint32_t)((col >> 3) * rows * 16 + row * 16 + ((col & 7) << 1));
}

__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b) {
  return (uint32_t)__bfloat16_as_ushort(a) | ((uint32_t)__bfloat16_as_ushort(b) << 16);
}

// The pieces of two neighbouring values, written to columns col, col + 1 of a tile.  A value
// that is not finite keeps its first piece (the rest would be NaN from inf - inf).
template <int P>
__device__ __forceinline__ void put2(unsigned char* tile, int rows, int pcols, int row, int col, float a, float b) {
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const __nv_bfloat16 ha = __float2bfloat16_rn(a), hb = __float2bfloat16_rn(b);
    *reinterpret_cast<uint32_t*>(tile + tile_off(rows, row, p * pcols + col)) = pack2(ha, hb);
    if (p + 1 < P) {
      a -= __bfloat162float(ha);
      b -= __bfloat162float(hb);
      if (p == 0) {
        if (!(fabsf(a) <= 3.4e38f)) a = 0.f;
        if (!(fabsf(b) <= 3.4e38f)) b = 0.f;
      }
    }
  }
}

__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A lane's ldmatrix address is a constant part and a part that the step of k (or the piece and the column
// group) moves: 16-byte units of a swizzled row are XORed, everything else is added.
template <bool U>
struct LaneAddr {
  uint32_t base;   // of the lane's row and unit
  int rows;
  __device__ __forceinline__ LaneAddr(const unsigned char* tile, int rows_, int row, int unit) : rows(rows_) {
    base = s_addr(tile) + (U ? unit * rows * 16 + row * 16 : row * 128 + ((unit ^ (row & 7)) << 4));
  }
  // `col` more columns (a multiple of 8 that shares no bit with the unit), `row` more rows (of 8)
  __device__ __forceinline__ uint32_t at(int row, int col) const {
    if (U) return base + (col >> 3) * rows * 16 + row * 16;
    return ((base + (col >> 6) * rows * 128 + row * 128) ^ ((col & 63) << 1));
  }
};

// acc (16 x 8 NT) += A[m0 .. m0+15][k0 .. k1) B[k0 .. k1)[n0 .. n0 + 8 NT).
// AT: A is stored with k along the rows; BT: B is stored with k along the rows (otherwise n).
// AU / BU: A / B is a tile of the recurrences (unit_off).
// PA / PB pieces lie apc / bpc columns apart; products of pieces i + j >= PM are dropped
// (PM is the piece count of the fp32 operands: what is dropped is below their own rounding).
// One warp; k0, k1 multiples of 16, NT even.  Fragment layout of m16n8k16: lane 4 g + t holds
// rows g and g + 8, columns 2 t and 2 t + 1 of each 16 x 8 block of acc.
template <int NT, bool AT, bool BT, int PA, int PB, int PM, bool AU = false, bool BU = false>
__device__ __forceinline__ void mma_tile(float (&acc)[NT][4], const unsigned char* A, int arows, int apc, int m0,
                                         const unsigned char* B, int brows, int bpc, int n0, int k0, int k1) {
  const int lane = threadIdx.x & 31;
  const LaneAddr<AU> a_at(A, arows, AT ? (lane & 7) + ((lane >> 4) & 1) * 8 : m0 + (lane & 15),
                          AT ? (lane >> 3) & 1 : lane >> 4);
  const LaneAddr<BU> b_at(B, brows, BT ? lane & 15 : n0 + (lane & 7) + ((lane >> 4) & 1) * 8,
                          BT ? lane >> 4 : (lane >> 3) & 1);
  // Tensor-core sums truncate: where three pieces promise fp32 accuracy, two steps of k are summed
  // apart and added in fp32 (48 truncating additions to one sum left dk 1.7e-6 off).
  constexpr bool kApart = PM == 3;
  float part[kApart ? NT : 1][4];
#pragma unroll 2
  for (int k = k0; k < k1; k += 16) {
    if (kApart && ((k - k0) & 16) == 0) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[kApart ? j : 0][i] = 0.f;
    }
    uint32_t a[PA][4];
#pragma unroll
    for (int p = 0; p < PA; ++p) {
      if (AT) ldsm4t(a[p], a_at.at(k, p * apc + m0));
      else ldsm4(a[p], a_at.at(0, p * apc + k));
    }
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
#pragma unroll
      for (int q = 0; q < PB; ++q) {
        uint32_t b[4];
        if (BT) ldsm4t(b, b_at.at(k, q * bpc + n0 + 8 * j));
        else ldsm4(b, b_at.at(8 * j, q * bpc + k));
#pragma unroll
        for (int p = 0; p < PA; ++p) {
          if (p + q < PM) {
            mma16816(kApart ? part[kApart ? j : 0] : acc[j], a[p], b[0], b[1]);
            mma16816(kApart ? part[kApart ? j + 1 : 0] : acc[j + 1], a[p], b[2], b[3]);
          }
        }
      }
    }
    if (kApart && (((k - k0) & 16) != 0 || k + 16 >= k1)) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] += part[kApart ? j : 0][i];
    }
  }
}

template <int NT>
__device__ __forceinline__ void zero(float (&a)[NT][4]) {
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) a[j][i] = 0.f;
}

// ---- asynchronous copies ----
__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Copies `bytes` (a multiple of 16) with all threads of the block.
__device__ __forceinline__ void cp_tile(unsigned char* dst, const unsigned char* src, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) cp16(dst + i, src + i);
}

// ---- where a chunk lies ----
struct Chunk {
  int seq, idx, len;   // sequence, chunk within it, tokens in it (0: no such chunk)
  int64_t b, t0;       // batch row and first token
};

// Token range of sequence s, clamped to the tensors, so that wrong offsets cannot reach outside.
__device__ __forceinline__ void seq_range(const Params& p, int s, int64_t& b, int64_t& t0, int64_t& n) {
  if (p.offsets == nullptr) {
    b = s;
    t0 = 0;
    n = p.time;
    return;
  }
  b = 0;
  const int64_t lo = p.offsets[s], hi = p.offsets[s + 1];
  t0 = lo < 0 ? 0 : (lo > p.time ? p.time : lo);
  const int64_t e = hi < t0 ? t0 : (hi > p.time ? p.time : hi);
  n = e - t0;
}

// First chunk slot and chunk count of sequence s (packed: as far as the slots go).
__device__ __forceinline__ void seq_slots(const Params& p, int s, int& c0, int& nc) {
  if (p.offsets == nullptr) {
    c0 = s * p.nchunk;
    nc = p.nchunk;
  } else {
    c0 = p.cstart[s];
    nc = p.cstart[s + 1] - c0;
  }
}

__device__ __forceinline__ Chunk chunk_at(const Params& p, int c) {
  Chunk r;
  if (p.offsets == nullptr) {
    r.seq = c / p.nchunk;
    r.idx = c - r.seq * p.nchunk;
  } else {
    if (c >= p.cstart[p.nseq]) {
      r.seq = -1;
      r.idx = c - p.cstart[p.nseq];
      r.len = 0;
      r.b = 0;
      r.t0 = 0;
      return r;
    }
    int lo = 0, hi = p.nseq;   // the last s with cstart[s] <= c
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (p.cstart[m] <= c) lo = m;
      else hi = m;
    }
    r.seq = lo;
    r.idx = c - p.cstart[lo];
  }
  int64_t t0, n;
  seq_range(p, r.seq, r.b, t0, n);
  r.t0 = t0 + (int64_t)r.idx * kChunk;
  const int64_t left = n - (int64_t)r.idx * kChunk;
  r.len = (int)(left < kChunk ? (left < 0 ? 0 : left) : kChunk);
  return r;
}

// The stretch of a sequence that a block of the recurrences walks: all of it, or one segment.
struct Span {
  int seq, g, g0, slot0, nc;   // g: segment; g0: the sequence's first; slot0, nc: chunks (nc < 0: no such segment)
  int64_t b, t0, n;
  bool first, last;
};

template <bool CUT = true>
__device__ __forceinline__ Span span_at(const Params& p, int turn) {
  Span s;
  int j = 0, ns = 1, total;
  s.g = turn;
  if (!CUT || p.seg == 0) {
    s.seq = p.offsets != nullptr ? p.order[turn] : turn;   // the longest sequences start first
  } else if (p.offsets == nullptr) {
    ns = max(1, (p.nchunk + p.seg - 1) / p.seg);
    s.seq = turn / ns;
    j = turn - s.seq * ns;
  } else {
    if (turn >= p.segstart[p.nseq]) {
      s.nc = -1;
      return s;
    }
    int lo = 0, hi = p.nseq;   // the last sequence whose first segment is not behind turn
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (p.segstart[m] <= turn) lo = m;
      else hi = m;
    }
    s.seq = lo;
    j = turn - p.segstart[lo];
    ns = p.segstart[lo + 1] - p.segstart[lo];
  }
  seq_range(p, s.seq, s.b, s.t0, s.n);
  seq_slots(p, s.seq, s.slot0, total);
  s.first = j == 0;
  s.last = j == ns - 1;
  s.g0 = turn - j;
  s.nc = total;
  if (CUT && p.seg > 0) {
    const int c0 = j * p.seg;
    s.slot0 += c0;
    s.t0 += (int64_t)c0 * kChunk;
    s.nc = min(p.seg, total - c0);
    s.n = min(s.n - (int64_t)c0 * kChunk, (int64_t)s.nc * kChunk);
  }
  return s;
}

__device__ __forceinline__ size_t slot_head(const Params& p, int c, int h) { return (size_t)c * p.hv + h; }

// One chunk's dbeta and dg from the sums the recurrences left: a warp, two tokens a lane.
__device__ __forceinline__ void gate_sums(const Params& p, const Chunk& ch, size_t at, int h, int lane) {
  float x[2] = {0.f, 0.f}, db[2] = {0.f, 0.f}, sds = 0.f;
  for (int n = 0; n < p.nv; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const size_t i = (at * p.nv + n) * kChunk + 2 * lane + e;
      x[e] += p.odo[i] - p.vdv[i];
      db[e] += p.edu[i];
    }
  for (int i = lane; i < 4 * p.nv; i += 32) sds += p.sds[at * p.nv * 4 + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sds += __shfl_xor_sync(0xffffffffu, sds, o);
  float s = x[0] + x[1];             // suffix sums
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float y = __shfl_down_sync(0xffffffffu, s, o);
    if (lane + o < 32) s += y;
  }
  const int64_t to = (ch.b * p.time + ch.t0 + 2 * lane) * p.hv + h;
  if (2 * lane < ch.len) {
    p.dg[to] = s + sds;
    p.dbeta[to] = db[0];
  }
  if (2 * lane + 1 < ch.len) {
    p.dg[to + p.hv] = s - x[0] + sds;
    p.dbeta[to + p.hv] = db[1];
  }
}

// ---- launchers ----
cudaError_t launch_plan(const Params& p, cudaStream_t s);
cudaError_t launch_prep(const Params& p, int dtype, cudaStream_t s);
cudaError_t launch_scan(const Params& p, int dtype, bool state_only, cudaStream_t s);
cudaError_t launch_rscan(const Params& p, int dtype, bool state_only, cudaStream_t s);
cudaError_t launch_join(const Params& p, cudaStream_t s);
cudaError_t launch_grad(const Params& p, int dtype, cudaStream_t s);
template <typename T>
cudaError_t launch_grad_tc(const Params& p, cudaStream_t s);
// The gradients of 16-bit inputs go through tcgen05, whose shared memory two pieces of every tile fill
// (4 x 2048 tokens, 16 heads of 128 x 128, bf16: 120 us against 292 with mma.sync).
constexpr bool grad_on_tc(int dtype) { return dtype != 0; }
cudaError_t launch_step(const qrb_delta_step_args& a, cudaStream_t s);

}  // namespace delta
}  // namespace qrb
