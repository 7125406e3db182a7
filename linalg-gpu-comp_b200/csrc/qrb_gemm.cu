// y = epilogue(A B^T) on the 5th-generation tensor cores: the linear layer's forward product
// (x w^T with bias, activation and residual in the epilogue) and both products of its backward.
//
// Persistent warp-specialised blocks, one per SM: a TMA producer fills a ring of 64-deep stages
// (128-byte swizzle; operands with k along their rows and operands with k across them are both
// read as they lie, so no backward product transposes anything), one thread issues MMAs 16 deep into
// TMEM, and eight warps run the epilogue of one tile while the next one's MMAs fill the other
// accumulator buffer.
//   * Large outputs: pairs of blocks (cta_group::2) on 256 x 256 tiles, each block loading 128 rows of
//     A and 128 of B: 32 KB per 512 cycles of MMAs.  One block on 128 x 256 needs 48 KB for the same
//     time, more than L2 delivers to every SM at once (4096 x 2048 x 8192 took twice its MMA time).
//   * Smaller ones: single blocks on 128 x 128 or 64 tiles.
//   * Few rows (m <= 128): the operands change places, so the 128-row side of the MMA is the weight
//     and its 64 or 128 column side the rows: no tensor-core row is wasted on padding, and the
//     weight streams through once.
//   * Few tiles: the blocks divide k; fp32 partials are added in order by reduce_kernel, which
//     then runs the epilogue, so results repeat.
//   * Long k: the tensor cores' accumulation truncates, one-sidedly, so its bias grows with the number of
//     additions (16 products each): 1.0e-7 of a sum of one sign each, 6.7e-3 of one of 2^20 rows, where
//     rounding to bf16 is at most 3.9e-3 off.  k is cut, as for few tiles, where that bias would pass a
//     half of the output's rounding.
//   * fp32: three bf16 planes per operand, x = x0 + x1 + x2 to 2^-27; the six products x_i w_j with
//     i + j < 3.  The five small ones have an accumulator of their own, and k is cut at 512 (fp32
//     partials beyond): the tensor cores' accumulation truncates, and its bias grows with the
//     number of additions to the large sum (k = 1432 in one piece was 1.5e-6 off).
//
// Every wait is bounded (mbar_wait_abort); see qrb_wide.cu.  No TMA load uses cluster multicast.
#include "qrb_gemm.cuh"

#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "qrb_sm100.cuh"

namespace qrb {
namespace gemm {
namespace {

using namespace sm100;

constexpr int kBM = 128, kBK = 64, kThreads = 384;   // warps: producer, MMA, 2 idle, 8 epilogue
constexpr int kMaxTerms = 6;
// Longest k of one accumulation.  fp32: see the head of this file.  16 bits: 2^18 / 16 additions leave up to
// 1.7e-3, less than half of bf16's eps / 2 = 3.9e-3; 2^15 / 16 leave 2.1e-4 of fp16's 4.9e-4.
constexpr int64_t kMaxSplitK32 = 512, kMaxSplitBf16 = 1 << 18, kMaxSplitF16 = 1 << 15;

struct GemmArgs {
  int64_t M, N;                 // MMA orientation: A's rows, B's rows
  int tiles_m, tiles_n, splits;
  int kblocks, per_split;       // 64-deep blocks of k in all and per split
  int terms, sets;              // piece products; accumulators per tile (2: small products apart)
  int a_mn, b_mn, swap;         // swap: A's rows are the output's columns
  uint32_t idesc;
  signed char pa[kMaxTerms], pb[kMaxTerms], set[kMaxTerms];
  float* partial;               // splits > 1: [split][m][n] of the output
  int64_t out_m, out_n;
  Epilogue e;
  int* err;
};

template <int BN, bool PAIR>
struct Cfg {
  static constexpr int kRowsB = PAIR ? BN / 2 : BN;   // rows of B this block loads
  static constexpr uint32_t kA = kBM * kBK * 2, kB = kRowsB * kBK * 2, kStage = kA + kB;
  static constexpr uint32_t kTurn = 8 * 32 * 33 * 4;   // a 32 x 32 tile for each epilogue warp to turn
  static constexpr int kStages = kStage > 24576 ? 5 : 6;
  static constexpr uint32_t kBar = kStages * kStage;
  static constexpr uint32_t kOffTurn = kBar + 256;
  static constexpr uint32_t kSmem = kOffTurn + kTurn + 1024;
  static_assert(kSmem <= 232448, "shared memory of one block");
};

struct Bars {
  uint64_t full[6], empty[6], accf[2], acce[2], drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Bars) <= 256, "barrier block");

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int dtype) {
  if (dtype == QRB_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight neighbouring fp32 outputs of a 16-byte aligned row, the first `count` of which exist.
__device__ __forceinline__ void store8(void* p, int64_t i, const float* x, int count) {
  float* to = static_cast<float*>(p) + i;
  if (count == 8) {
    reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < count) to[j] = x[j];
}

__device__ __forceinline__ void add8(const void* p, int64_t i, int dtype, float* x, int count) {
  if (count == 8 && dtype != QRB_F32) {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (dtype == QRB_BF16) {
        x[2 * j] += __uint_as_float(u[j] << 16);
        x[2 * j + 1] += __uint_as_float(u[j] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
        x[2 * j] += f.x;
        x[2 * j + 1] += f.y;
      }
    }
    return;
  }
  if (count <= 0) return;
  float y[8];   // all loads first: one under a condition would be waited for before the next
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = load1(p, i + min(j, count - 1), dtype);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] += y[j];
}

__device__ __forceinline__ bool aligned_rows(const void* p, int64_t ld, int dtype) {
  const int64_t v = dtype == QRB_F32 ? 4 : 8;
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % v == 0;
}

// Work unit u: split fastest (the splits of a tile run together), then tiles in groups of eight
// rows of tiles, so that blocks running together share operand tiles in L2.
__device__ __forceinline__ void tile_of(const GemmArgs& g, int u, int& tm, int& tn, int& sp) {
  sp = u % g.splits;
  const int t = u / g.splits;
  const int group = 8 * g.tiles_n, gi = t / group, first = gi * 8;
  const int rows = min(8, g.tiles_m - first), r = t - gi * group;
  tm = first + r % rows;
  tn = r / rows;
}

template <int BN, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            const __grid_constant__ GemmArgs g) {
  using C = Cfg<BN, PAIR>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                       ~uintptr_t(1023));
  Bars& bars = *reinterpret_cast<Bars*>(sm + C::kBar);
  volatile int* abort = &bars.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int units = g.tiles_m * g.tiles_n * g.splits;
  const int bufs = 2 * g.sets * BN <= 512 ? 2 : 1;
  const uint32_t cols = (uint32_t)(bufs * g.sets * BN);   // a power of two, at least 128

  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.accf[i], 1);
      mbar_init(&bars.acce[i], PAIR ? 16 : 8);
    }
    mbar_init(&bars.drain, 1);
    bars.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if (PAIR) tmem_alloc_pair(&bars.tmem, cols);
    else tmem_alloc(&bars.tmem, cols);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();   // the peer's barriers exist
  tc_fence_after();
  const uint32_t tmem = bars.tmem;

  if (warp == 0) {
    // ---------------- TMA producer (both blocks of a pair, for the leader's barriers) ----------------
    if (lane == 0) {
      prefetch_tensormap(&map_a);
      prefetch_tensormap(&map_b);
      int64_t it = 0;
      bool ok = true;
      for (int u = first; u < units && ok; u += step) {
        int tm, tn, sp;
        tile_of(g, u, tm, tn, sp);
        const int row = (PAIR ? 2 * tm + rank : tm) * kBM, col = tn * BN + rank * C::kRowsB;
        const int kb0 = sp * g.per_split, kb1 = min(g.kblocks, kb0 + g.per_split);
        for (int t = 0; t < g.terms && ok; ++t)
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int st = (int)(it % C::kStages);
            const int64_t use = it / C::kStages;
            if (use > 0 && !mbar_wait_abort(&bars.empty[st], (uint32_t)((use - 1) & 1), abort, g.err, 41)) {
              ok = false;
              break;
            }
            unsigned char* sa = sm + st * C::kStage;
            unsigned char* sb = sa + C::kA;
            if (rank == 0) mbar_arrive_expect_tx(&bars.full[st], (PAIR ? 2 : 1) * C::kStage);
            const uint32_t bar = PAIR ? mapa_shared(smem_u32(&bars.full[st]), 0) : 0;
            auto load = [&](void* dst, const CUtensorMap* map, int x, int y, int z) {
              if (PAIR) tma_load_3d_pair(dst, map, x, y, z, bar);
              else tma_load_3d(dst, map, x, y, z, &bars.full[st]);
            };
            if (g.a_mn) {
              load(sa, &map_a, row, kb * kBK, g.pa[t]);
              load(sa + 8192, &map_a, row + 64, kb * kBK, g.pa[t]);
            } else {
              load(sa, &map_a, kb * kBK, row, g.pa[t]);
            }
            if (g.b_mn) {
              for (int j = 0; j < C::kRowsB / 64; ++j) load(sb + j * 8192, &map_b, col + 64 * j, kb * kBK, g.pb[t]);
            } else {
              load(sb, &map_b, kb * kBK, col, g.pb[t]);
            }
          }
      }
      if (*abort && rank == 0) {   // every load issued must land before the shared memory goes away
        for (int st = 0; st < C::kStages; ++st)
          if (it > st) mbar_wait(&bars.full[st], (uint32_t)(((it - 1 - st) / C::kStages) & 1), 1u << 22);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the leader of a pair) ----------------
    if (lane == 0 && rank == 0) {
      int64_t it = 0;
      int n = 0;
      bool ok = true, issued = false;
      auto commit = [&](uint64_t* bar) {
        if (PAIR) mma_commit_pair(bar);
        else mma_commit(bar);
      };
      const uint32_t a_lbo = g.a_mn ? 8192 : 16, a_step = g.a_mn ? 2048 : 32;
      const uint32_t b_lbo = g.b_mn ? 8192 : 16, b_step = g.b_mn ? 2048 : 32;
      for (int u = first; u < units && ok; u += step, ++n) {
        int tm, tn, sp;
        tile_of(g, u, tm, tn, sp);
        const int kb0 = sp * g.per_split, kb1 = min(g.kblocks, kb0 + g.per_split);
        const int buf = n % bufs, use = n / bufs;
        if (use > 0 && !mbar_wait_abort(&bars.acce[buf], (uint32_t)((use - 1) & 1), abort, g.err, 42)) break;
        tc_fence_after();
        int seen = 0;   // accumulators that hold something already
        for (int t = 0; t < g.terms && ok; ++t) {
          const uint32_t d = tmem + (uint32_t)((buf * g.sets + g.set[t]) * BN);
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int st = (int)(it % C::kStages);
            if (!mbar_wait_abort(&bars.full[st], (uint32_t)((it / C::kStages) & 1), abort, g.err, 43)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_u32(sm + st * C::kStage), sb = sa + C::kA;
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk) {
              const uint64_t ad = sdesc_sw128(sa + kk * a_step, a_lbo, 1024), bd = sdesc_sw128(sb + kk * b_step, b_lbo, 1024);
              const uint32_t acc = ((seen >> g.set[t]) & 1) | (kk > 0);
              if (PAIR) mma_f16_pair(d, ad, bd, g.idesc, acc);
              else mma_f16(d, ad, bd, g.idesc, acc);
            }
            seen |= 1 << g.set[t];
            commit(&bars.empty[st]);
            issued = true;
          }
        }
        if (ok) commit(&bars.accf[buf]);
      }
      if (*abort && issued) {   // tensor memory must not be released under running MMAs
        mma_commit(&bars.drain);
        mbar_wait(&bars.drain, 0, 1u << 22);
      }
    }
  } else if (warp >= 4) {
    // ---------------- epilogue: TMEM lane = A's row, half of the columns a warp ----------------
    const int q = warp & 3, c_first = ((warp - 4) >> 2) * (BN / 2), c_last = c_first + BN / 2;
    const uint32_t tl = (uint32_t)(32 * q) << 16;
    float* turned = reinterpret_cast<float*>(sm + C::kOffTurn) + (warp - 4) * 32 * 33;
    const Epilogue& e = g.e;
    const bool vec = (e.y == nullptr || aligned_rows(e.y, e.ldy, e.dtype)) &&
                     (e.residual == nullptr || aligned_rows(e.residual, e.ldr, e.dtype)) &&
                     (e.pre == nullptr || aligned_rows(e.pre, e.ldpre, e.dtype));
    int n = 0;
    for (int u = first; u < units; u += step, ++n) {
      int tm, tn, sp;
      tile_of(g, u, tm, tn, sp);
      const int buf = n % bufs, use = n / bufs;
      const int64_t r = (int64_t)(PAIR ? 2 * tm + rank : tm) * kBM + 32 * q + lane, c0 = (int64_t)tn * BN;
      const float rb = g.swap && e.bias != nullptr && r < g.M ? load1(e.bias, r, e.dtype) : 0.f;
      // the whole warp goes on or leaves: tensor memory loads are collective
      if (!__all_sync(0xffffffffu, mbar_wait_abort(&bars.accf[buf], (uint32_t)(use & 1), abort, g.err, 44))) break;
      tc_fence_after();
#pragma unroll 1
      for (int c = c_first; c < c_last; c += 32) {
        // lane j holds the bias of column c + j
        const float cb = !g.swap && g.splits == 1 && e.bias != nullptr
                             ? load1(e.bias, min(c0 + c + lane, g.N - 1), e.dtype) : 0.f;
        float x[32];
        const uint32_t at = tmem + tl + (uint32_t)(buf * g.sets * BN + c);
        tmem_ld32(at, x);
        if (g.sets == 2) {
          float y[32];
          tmem_ld32(at + BN, y);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (fabsf(x[j]) <= 3.4e38f) x[j] += y[j];   // inf * 0 among the small products is no NaN of the sum
        }
        if (c + 32 >= c_last) {   // this warp's last read of the buffer
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR) mbar_arrive_cluster(mapa_shared(smem_u32(&bars.acce[buf]), 0));
            else mbar_arrive(&bars.acce[buf]);
          }
        }
        if (!g.swap && g.splits == 1 && e.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] += __shfl_sync(0xffffffffu, cb, j);
        }
        if (g.splits == 1 && !g.swap && !vec) {
          // rows that are not 16-byte aligned: a lane's row written value by value would touch 32 rows an
          // instruction, so the warp turns the tile and writes 32 neighbouring columns of one row at a time
          const int rows = (int)max((int64_t)0, min((int64_t)32, g.M - (r - lane)));
          const bool mine = c0 + c + lane < g.N;
          auto turn = [&] {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) turned[lane * 33 + j] = x[j];
            __syncwarp();
          };
          const int64_t row = r - lane, cc = c0 + c + lane;
          if (e.pre != nullptr) {
            turn();
            if (mine)
              for (int i = 0; i < rows; ++i) store1(e.pre, (row + i) * e.ldpre + cc, e.dtype, turned[i * 33 + lane]);
          }
          activate_all(x, e.act);
          turn();
          if (mine) {
            for (int i = 0; i < rows; i += 8) {
              float add[8];
#pragma unroll
              for (int u = 0; u < 8; ++u)
                add[u] = e.residual != nullptr ? load1(e.residual, (row + min(i + u, rows - 1)) * e.ldr + cc, e.dtype) : 0.f;
#pragma unroll
              for (int u = 0; u < 8; ++u)
                if (i + u < rows) store1(e.y, (row + i + u) * e.ldy + cc, e.dtype, turned[(i + u) * 33 + lane] + add[u]);
            }
          }
          continue;
        }
        if (g.splits == 1 && !g.swap && e.dtype != QRB_F32) {
          // Aligned 16-bit rows: the warp passes its 32 x 32 values through shared memory (64-byte rows, units
          // of 16 bytes XORed so that both directions are free of bank conflicts), and four lanes hold 64
          // neighbouring bytes of a row in place of one lane 16 (4096 x 512 x 8192: 47.8 -> 43.7 us).
          const int64_t row0 = r - lane, left = g.N - (c0 + c) - 8 * (lane & 3), cc = c0 + c + 8 * (lane & 3);
          unsigned char* buf = reinterpret_cast<unsigned char*>(turned);
          auto own = [&](int u) { return reinterpret_cast<uint4*>(buf + lane * 64 + ((u ^ (lane >> 1)) & 3) * 16); };
          auto far = [&](int i) {   // row 8 i + lane / 4
            const int rr = 8 * i + (lane >> 2);
            return reinterpret_cast<uint4*>(buf + rr * 64 + ((lane ^ (rr >> 1)) & 3) * 16);
          };
          auto put = [&](void* to, int64_t ld) {
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u)
              *own(u) = make_uint4(pack16(x[8 * u], x[8 * u + 1], e.dtype), pack16(x[8 * u + 2], x[8 * u + 3], e.dtype),
                                   pack16(x[8 * u + 4], x[8 * u + 5], e.dtype), pack16(x[8 * u + 6], x[8 * u + 7], e.dtype));
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int64_t row = row0 + 8 * i + (lane >> 2);
              uint16_t* at = static_cast<uint16_t*>(to) + row * ld + cc;
              if (row >= g.M) continue;
              if (left >= 8) {
                *reinterpret_cast<uint4*>(at) = *far(i);
              } else {
                for (int j = 0; j < left; ++j) at[j] = reinterpret_cast<const uint16_t*>(far(i))[j];
              }
            }
          };
          if (e.pre != nullptr) put(e.pre, e.ldpre);
          activate_all(x, e.act);
          if (e.residual != nullptr) {
            const int64_t at = min(r, g.M - 1) * e.ldr + c0 + c, n32 = g.N - (c0 + c);
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              add8(e.residual, at + j, e.dtype, x + j, (int)max((int64_t)0, min((int64_t)8, n32 - j)));
          }
          put(e.y, e.ldy);
          continue;
        }
        if (r >= g.M) continue;
        if (g.splits > 1) {
          if (g.swap) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c0 + c + j < g.N) g.partial[((int64_t)sp * g.out_m + c0 + c + j) * g.out_n + r] = x[j];
          } else {
            float* to = g.partial + ((int64_t)sp * g.out_m + r) * g.out_n + c0 + c;
            const bool v4 = g.out_n % 4 == 0;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              if (v4 && c0 + c + j + 3 < g.N) *reinterpret_cast<float4*>(to + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
              else
                for (int i = 0; i < 4; ++i)
                  if (c0 + c + j + i < g.N) to[j + i] = x[j + i];
            }
          }
          continue;
        }
        if (g.swap) {
          const int count = (int)min((int64_t)32, g.N - (c0 + c));
          if (count <= 0) continue;
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] += rb;
          if (e.pre != nullptr)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < count) store1(e.pre, (c0 + c + j) * e.ldpre + r, e.dtype, x[j]);
          activate_all(x, e.act);
          if (e.residual != nullptr)
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] += load1(e.residual, (c0 + c + min(j, count - 1)) * e.ldr + r, e.dtype);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < count) store1(e.y, (c0 + c + j) * e.ldy + r, e.dtype, x[j]);
          continue;
        }
        const int64_t left = g.N - (c0 + c);
        if (e.pre != nullptr)
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            store8(e.pre, r * e.ldpre + c0 + c + j, x + j, (int)max((int64_t)0, min((int64_t)8, left - j)));
        activate_all(x, e.act);
        if (e.residual != nullptr)
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            add8(e.residual, r * e.ldr + c0 + c + j, e.dtype, x + j, (int)max((int64_t)0, min((int64_t)8, left - j)));
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          store8(e.y, r * e.ldy + c0 + c + j, x + j, (int)max((int64_t)0, min((int64_t)8, left - j)));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();   // neither block leaves while the other may still reach its memory
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem, cols);
    else tmem_dealloc(tmem, cols);
  }
}

// y = epilogue(sum of the splits' partials, in order).
__global__ void __launch_bounds__(256) reduce_kernel(const float* part, int splits, int64_t m, int64_t n, Epilogue e) {
  const int64_t total = m * n, c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  const float b = e.bias != nullptr ? load1(e.bias, c, e.dtype) : 0.f;
  for (int64_t r = blockIdx.y; r < m; r += gridDim.y) {
    float x = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) x += part[s * total + r * n + c];
    x += b;
    if (e.pre != nullptr) store1(e.pre, r * e.ldpre + c, e.dtype, x);
    x = activate(x, e.act);
    if (e.residual != nullptr) x += load1(e.residual, r * e.ldr + c, e.dtype);
    store1(e.y, r * e.ldy + c, e.dtype, x);
  }
}

// ---- host side ----
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

bool make_map(CUtensorMap* map, const Operand& o, int64_t mn, int64_t k, bool half, int rows) {
  auto fn = encoder();
  if (fn == nullptr) return false;
  const uint64_t inner = (uint64_t)(o.mn_major ? mn : k), outer = (uint64_t)(o.mn_major ? k : mn);
  cuuint64_t dims[3] = {inner, outer, (cuuint64_t)o.pieces};
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.pieces > 1 ? o.plane : o.ld * (int64_t)outer) * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)(o.mn_major ? kBK : rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p),
            dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
  int bn, swap, pair, tiles_m, tiles_n, splits, kblocks, per_split;
};

// Tile shape and split of an m x n x k product.  Up to 128 rows: swapped, the narrowest tile that
// holds them.  Otherwise pairs on 256 x 256 where these fill two thirds of the SMs (or nearly: the
// last, partly filled wave counts), else single blocks on 128 x 128 where these do (a wide tile reads the
// least shared memory per MMA, an idle SM costs more), else on 128 x 64; where even those leave half of the
// SMs idle, k is split.  (Blocks on 128 x 256 are at most twice the pairs, so they never fill two thirds
// where pairs do not fill one.)
Plan plan(int64_t m, int64_t n, int64_t k, int pieces, bool half) {
  Plan p{};
  const int sms = sm_count();
  p.kblocks = (int)((k + kBK - 1) / kBK);
  p.swap = m <= 128;
  auto tiles = [&](int bn, int pair) {
    p.bn = bn;
    p.pair = pair;
    p.tiles_m = (int)(((p.swap ? n : m) + kBM * (1 + pair) - 1) / (kBM * (1 + pair)));
    p.tiles_n = (int)(((p.swap ? m : n) + bn - 1) / bn);
    return (int64_t)p.tiles_m * p.tiles_n;
  };
  int64_t t;
  if (p.swap) {
    t = tiles(m <= 64 ? 64 : 128, 0);
  } else {
    t = tiles(256, 1);
    if (t * 3 < sms) t = tiles(128, 0);
    if (!p.pair && t * 3 < sms * 2) t = tiles(64, 0);
  }
  // a split is worth at least four stages of work, and there are 16 at most
  int64_t splits = !p.pair && t * 2 <= sms ? sms / t : 1;
  if (splits > (p.kblocks + 3) / 4) splits = (p.kblocks + 3) / 4;
  if (splits > 16) splits = 16;
  if (splits < 1) splits = 1;
  const int64_t longest = (pieces > 1 ? kMaxSplitK32 : half ? kMaxSplitF16 : kMaxSplitBf16) / kBK;
  const int64_t need = (p.kblocks + longest - 1) / longest;
  if (splits < need) splits = need;
  p.per_split = (int)((p.kblocks + splits - 1) / splits);
  p.splits = (p.kblocks + p.per_split - 1) / p.per_split;
  return p;
}

template <int BN, bool PAIR>
cudaError_t run(const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& g, cudaStream_t s) {
  constexpr int smem = Cfg<BN, PAIR>::kSmem;
  cudaError_t e = allow_smem<gemm_kernel<BN, PAIR>>(smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  const int sms = PAIR ? sm_count() / 2 : sm_count(), grid = (int)(units < sms ? units : sms);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(PAIR ? 2 * grid : grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, gemm_kernel<BN, PAIR>, ma, mb, g);
}

}  // namespace

bool supported() { return encoder() != nullptr; }

size_t scratch(int64_t m, int64_t n, int64_t k, int pieces, bool half) {
  if (m < 1 || n < 1 || k < 1) return 0;
  const Plan p = plan(m, n, k, pieces, half);
  return p.splits > 1 ? (size_t)p.splits * m * n : 0;
}

cudaError_t multiply(const Operand& A, const Operand& B, int64_t m, int64_t n, int64_t k, bool half, const Epilogue& e,
                     float* ws, cudaStream_t s) {
  const Plan p = plan(m, n, k, A.pieces, half);
  GemmArgs g{};
  const Operand &a = p.swap ? B : A, &b = p.swap ? A : B;
  g.M = p.swap ? n : m;
  g.N = p.swap ? m : n;
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.splits = p.splits;
  g.kblocks = p.kblocks;
  g.per_split = p.per_split;
  g.a_mn = a.mn_major;
  g.b_mn = b.mn_major;
  g.swap = p.swap;
  const uint32_t fmt = half ? 0 : 1;
  g.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a.mn_major << 15) | ((uint32_t)b.mn_major << 16) |
            ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)((p.pair ? 2 * kBM : kBM) >> 4) << 24);
  if (a.pieces == 1) {
    g.terms = 1;
    g.sets = 1;
  } else {   // smallest products first; the large one alone in accumulator 0
    static const signed char pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0}, set[6] = {1, 1, 1, 1, 1, 0};
    g.terms = 6;
    g.sets = 2;
    for (int i = 0; i < 6; ++i) {
      g.pa[i] = pa[i];
      g.pb[i] = pb[i];
      g.set[i] = set[i];
    }
  }
  g.partial = ws;
  g.out_m = m;
  g.out_n = n;
  g.e = e;
  g.err = device_error_flag();
  if (g.err == nullptr) return cudaErrorInvalidValue;
  CUtensorMap ma, mb;
  if (!make_map(&ma, a, g.M, k, half, kBM) || !make_map(&mb, b, g.N, k, half, p.pair ? p.bn / 2 : p.bn)) return cudaErrorInvalidValue;
  cudaError_t r;
  {
    const double bytes = (double)(m * k + n * k) * 2 * A.pieces + (double)m * n * (e.dtype == QRB_F32 ? 4 : 2);
    LaunchTimer t("linear_gemm_kernel", s, bytes, 2.0 * m * n * k);
    if (p.pair) r = run<256, true>(ma, mb, g, s);
    else if (p.bn == 64) r = run<64, false>(ma, mb, g, s);
    else r = run<128, false>(ma, mb, g, s);
  }
  if (r != cudaSuccess || p.splits == 1) return r;
  LaunchTimer t("linear_reduce_kernel", s, 4.0 * p.splits * m * n, (double)p.splits * m * n);
  reduce_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)(m < 1024 ? m : 1024)), 256, 0, s>>>(ws, p.splits, m, n, e);
  return cudaGetLastError();
}

}  // namespace gemm
}  // namespace qrb
