// Tensor-memory plumbing of the gated delta rule's recurrences (qrb_delta_scan.cu,
// qrb_delta_rscan.cu).
//
// Both recurrences work on transposed states: TMEM lane = value column, so a thread owns a value
// column from the state through u to the output, every accumulator it needs is in its own lane, and
// what it writes back (pieces of the state, of F, U, W) is the A operand of the next product without
// any exchange between threads.  The B operands are the chunk's tiles as prep_kernel laid them out:
// with k along their 128-byte rows (K-major) for products over dk or over a chunk's columns, and the
// same bytes read across the rows (MN-major) for their transposes.
#pragma once

#include "qrb_delta.cuh"
#include "qrb_sm100.cuh"

namespace qrb {
namespace delta {

using namespace sm100;

constexpr int kParts = 4;                   // threads that share a value column
constexpr int kTok = kChunk / kParts;       // tokens of a thread
// Two kernels that may run at the same time (their launches say so): the first lets the second start once
// all its blocks have, and the second does not end before the first has.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

constexpr int kIssuer = kLanes * kParts / 32, kLoader = kIssuer + 1;   // sixteen warps compute, one issues MMAs, one loads
constexpr int kTcThreads = 32 * (kLoader + 1);
constexpr int kSmemLimit = 232448;

// kind::f16, bf16 operands, fp32 accumulation, M = 128, A in tensor memory.
__host__ __device__ constexpr uint32_t idesc_bf16(int n, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void mma_bf16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// D (128 x N) (+)= A B over K, piece products i + j < PM, smallest first.
//   A in TMEM: piece i at a + i * a_piece, 8 columns per 16 of K.
//   B in shared memory: K-major tile (N rows of 64-column blocks): piece j starts at column
//   j * b_piece; or (B_MN) K rows of 64-column blocks of N columns.
template <int N, int K, bool B_MN, int PA, int PB, int PM>
__device__ __forceinline__ void mma_pieces(uint32_t d, uint32_t a, uint32_t a_piece, uint32_t b, uint32_t acc) {
  constexpr uint32_t idesc = idesc_bf16(N, B_MN);
  constexpr uint32_t rows = B_MN ? K : N;                       // rows of the tile
  constexpr uint32_t block = rows * 128;                        // one 64-column block of it
  constexpr uint32_t piece = block * ((B_MN ? N : K) / 64);     // one piece
#pragma unroll
  for (int s = PM - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < PA; ++i) {
      const int j = s - i;
      if (j < 0 || j >= PB) continue;
#pragma unroll
      for (int k = 0; k < K / 16; ++k) {
        const uint32_t off = B_MN ? k * 2048u : (k >> 2) * block + (k & 3) * 32u;
        mma_bf16_ta(d, a + i * a_piece + 8 * k, sdesc_sw128(b + j * piece + off, B_MN ? block : 16u, 1024), idesc, acc);
        acc = 1;
      }
    }
}

// N consecutive 32-bit columns of this thread's lane; warp-collective, see tmem_ld32.
__device__ __forceinline__ void ld_cols(uint32_t taddr, float (&v)[16]) {
  __syncwarp();
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void ld_cols(uint32_t taddr, float (&v)[32]) { tmem_ld32(taddr, v); }

// Stores; the caller waits with tmem_st_wait.
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&v)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&v)[8]) {
  __syncwarp();
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// One copy of contiguous global memory (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Brings contiguous global memory (the same alignment) into L2.
__device__ __forceinline__ void bulk_prefetch(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

constexpr uint32_t kNoTmem = 0xffffffffu;

// N values of this lane as PS pieces of N / 2 columns each, piece_cols apart.  KEEP > 0: the first KEEP
// pieces also go to a tile of the gradient kernel (32 value columns as rows, pieces of `cols` columns,
// written in units of 8).  One piece at a time: x becomes what is left.
template <int PS, int KEEP, int N>
__device__ __forceinline__ void put_pieces(uint32_t taddr, uint32_t piece_cols, float (&x)[N], unsigned char* tile = nullptr,
                                           int row = 0, int cols = 0, int col = 0) {
#pragma unroll
  for (int i = 0; i < PS; ++i) {
    uint32_t w[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(x[2 * j + 1]), "f"(x[2 * j]));
      if (i + 1 < PS) {
        x[2 * j] -= __uint_as_float(w[j] << 16);
        x[2 * j + 1] -= __uint_as_float(w[j] & 0xffff0000u);
      }
    }
    if (taddr != kNoTmem) st_cols(taddr + i * piece_cols, w);
    if (i < KEEP) {
#pragma unroll
      for (int j = 0; j < N / 2; j += 4)
        *reinterpret_cast<uint4*>(tile + unit_off(kTile, row, i * cols + col + 2 * j)) =
            make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
    }
  }
}

template <int PS, int N>
__device__ __forceinline__ void fetch_pieces(const unsigned char* tile, int row, int cols, int col, float (&x)[N]) {
  uint4 u[PS][N / 8];
#pragma unroll
  for (int i = 0; i < PS; ++i)
#pragma unroll
    for (int j = 0; j < N / 8; ++j)
      u[i][j] = *reinterpret_cast<const uint4*>(tile + unit_off(kTile, row, i * cols + col + 8 * j));
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = 0.f;
#pragma unroll
  for (int i = PS - 1; i >= 0; --i)
#pragma unroll
    for (int j = 0; j < N / 8; ++j) {
      const uint32_t w[4] = {u[i][j].x, u[i][j].y, u[i][j].z, u[i][j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[8 * j + 2 * e] += __uint_as_float(w[e] << 16);
        x[8 * j + 2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
      }
    }
}

// N rows of a dense state column: all loads are issued at once, from the last existing row where
// there are no more (rows r0 + count - 1 exists), because a load under a condition would be waited
// for before the next.
template <int N>
__device__ __forceinline__ void load_column(const float* p, int64_t stride, int count, bool on, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __ldg(p + (int64_t)min(i, count - 1) * stride);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = on && i < count ? x[i] : 0.f;
}
template <int N>
__device__ __forceinline__ void store_column(float* p, int64_t stride, int count, const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < count) p[i * stride] = x[i];
}

// A thread's tokens of its value column, from a staged tile (kLanes values a token).
template <typename T>
__device__ __forceinline__ void staged(const unsigned char* tile, int tok, int lane_col, float (&x)[kTok]) {
  const T* t = reinterpret_cast<const T*>(tile) + tok * kLanes + lane_col;
#pragma unroll
  for (int i = 0; i < kTok; ++i) x[i] = to_f(t[i * kLanes]);
}

// A thread's tokens of its value column, to rows `stride` apart; `count` of them exist.
template <typename T>
__device__ __forceinline__ void store_tokens(T* p, int64_t stride, int count, const float (&x)[kTok]) {
  if (count >= kTok) {
#pragma unroll
    for (int i = 0; i < kTok; ++i, p += stride) *p = from_f<T>(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kTok; ++i, p += stride)
      if (i < count) *p = from_f<T>(x[i]);
  }
}

// x[i] = x[i] * g[i] and the like, the per-token factors read four at a time.
struct Gates {
  const float4 *gam, *tail, *bet;
  const float* last;
  __device__ __forceinline__ Gates(const unsigned char* g, int tb)
      : gam(reinterpret_cast<const float4*>(g) + tb / 4),
        tail(reinterpret_cast<const float4*>(g) + (kChunk + tb) / 4),
        bet(reinterpret_cast<const float4*>(g) + (2 * kChunk + tb) / 4),
        last(reinterpret_cast<const float*>(g) + kChunk - 1) {}
};
template <typename F>
__device__ __forceinline__ void with_tokens(const float4* g, F f) {
#pragma unroll
  for (int i = 0; i < kTok; i += 4) {
    const float4 v = g[i / 4];
    f(i, v.x);
    f(i + 1, v.y);
    f(i + 2, v.z);
    f(i + 3, v.w);
  }
}

// Lanes 2 l and 2 l + 1 get the sum over the warp's lanes of their x[l].
__device__ __forceinline__ float sum_columns(float (&x)[kTok]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const bool up = lane & (2 * o);
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const float give = up ? x[j] : x[j + o], keep = up ? x[j + o] : x[j];
      x[j] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * o);
    }
  }
  return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 1);
}

// A bounded wait a whole warp takes or leaves together (tensor-memory accesses are collective).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait_abort(bar, parity, abort, err, code));
}

__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

}  // namespace delta
}  // namespace qrb
