// Joining the segments of long sequences (the gated delta rule on few heads).
//
// A chunk after another, one head of one sequence keeps one SM busy.  Where heads and sequences leave
// most SMs idle, a sequence is cut into segments that run side by side, twice: first for the state alone
// (scan_kernel and rscan_kernel in their state-only forms), from zero, with the segment's transition A
// beside it (the state that the identity becomes with v = 0, dk more columns); then, when this kernel has
// joined the borders,
//     S_{j+1} = A_j S_j + B_j   forward,     dS_j = A_j^T dS_{j+1} + C_j   backward,
// with the right state for everything else.  Two passes over 1/p of the chunks and p small products
// replace one over all of them.  A block owns 8 columns of one (sequence, head) and walks its segments in
// fp32: with wider blocks the products of the few that there are take longer than a step's latency.  The
// sum over the transition's columns is cut into 4 for the same reason; the next transition is on its way
// by cp.async: 1.6 us a segment of 128 x 128.
#include "qrb_delta.cuh"

namespace qrb {
namespace delta {
namespace {

constexpr int kCols = 8, kGroups = 4;   // columns of a block; parts of the sum over the transition's columns

template <int DKP>
struct JoinLayout {
  static constexpr int kAStride = DKP + 4;   // rows of A at different banks
  static constexpr int kA = DKP * kAStride * 4, kX = DKP * kCols * 4;
  static constexpr int kBytes = 2 * kA + kX + kGroups * kX;
  static constexpr int kThreads = kGroups * DKP * kCols / 16;
};

template <int DKP, bool BACK>
__device__ __forceinline__ void join(const Params& p, int block) {
  using L = JoinLayout<DKP>;
  extern __shared__ __align__(16) unsigned char sm[];
  float* X = reinterpret_cast<float*>(sm + 2 * L::kA);   // [row][column]
  float* parts = X + DKP * kCols;                        // [group][row][column]
  const int tid = threadIdx.x;
  const int pitch = (p.dv + kLanes - 1) / kLanes * kLanes, tiles = (p.dv + kCols - 1) / kCols;
  const int tile = block % tiles, sh = block / tiles, h = sh % p.hv, seq = sh / p.hv;
  int g0, ns;
  if (p.offsets == nullptr) {
    ns = max(1, (p.nchunk + p.seg - 1) / p.seg);
    g0 = seq * ns;
  } else {
    g0 = p.segstart[seq];
    ns = p.segstart[seq + 1] - g0;
  }
  const int steps = ns - 2;
  if (steps <= 0) return;
  // step i joins segment j: forward 1, 2, ..., backward ns - 2, ns - 3, ...
  auto segment = [&](int i) { return g0 + (BACK ? ns - 2 - i : 1 + i); };
  // the four columns of one row that this thread sums up in the end
  const int mine = tid * 4;
  float* S = (BACK ? p.seg_ds : p.seg_s) + (size_t)(mine / kCols) * pitch + tile * kCols + mine % kCols;
  auto border = [&](int g) { return reinterpret_cast<float4*>(S + ((size_t)g * p.hv + h) * DKP * pitch); };
  auto load = [&](int i) {
    const float* a = p.seg_a + ((size_t)segment(i) * p.hv + h) * DKP * DKP;
    float* to = reinterpret_cast<float*>(sm + (i & 1) * L::kA);
    for (int u = tid; u < DKP * DKP / 4; u += L::kThreads) {
      const int r = u / (DKP / 4), c = u % (DKP / 4) * 4;
      cp16(to + r * L::kAStride + c, a + r * DKP + c);
    }
    cp_commit();
  };
  auto add = [](float4& y, float a, const float4& x) {
    y.x = fmaf(a, x.x, y.x);
    y.y = fmaf(a, x.y, y.y);
    y.z = fmaf(a, x.z, y.z);
    y.w = fmaf(a, x.w, y.w);
  };
  // 4 x 4 products: columns c0 .., rows row(0 .. 3), over a quarter of the sum
  const int group = tid / (DKP * kCols / 16), t = tid % (DKP * kCols / 16), c0 = (t & 1) * 4, rt = t >> 1;
  auto row = [&](int e) { return BACK ? rt * 4 + e : rt + DKP / 4 * e; };
  load(0);
  *reinterpret_cast<float4*>(X + mine) = *border(segment(0) + (BACK ? 1 : 0));
  float4 next = *border(segment(0) + (BACK ? 0 : 1));
  for (int i = 0; i < steps; ++i) {
    float4* out = border(segment(i) + (BACK ? 0 : 1));
    float4 sum = next, s[4] = {};
    next = *border(segment(min(i + 1, steps - 1)) + (BACK ? 0 : 1));
    cp_wait_all();
    __syncthreads();
    if (i + 1 < steps) load(i + 1);
    const float* A = reinterpret_cast<const float*>(sm + (i & 1) * L::kA);
#pragma unroll 2
    for (int l = group * (DKP / kGroups); l < (group + 1) * (DKP / kGroups); l += 4) {
      float4 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const float4*>(X + (l + e) * kCols + c0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (BACK) {   // A^T: row l + e of A, columns row(0 .. 3)
          const float4 a = *reinterpret_cast<const float4*>(A + (l + e) * L::kAStride + row(0));
          add(s[0], a.x, x[e]);
          add(s[1], a.y, x[e]);
          add(s[2], a.z, x[e]);
          add(s[3], a.w, x[e]);
        } else {
          const float4 a = *reinterpret_cast<const float4*>(A + row(e) * L::kAStride + l);
          add(s[e], a.x, x[0]);
          add(s[e], a.y, x[1]);
          add(s[e], a.z, x[2]);
          add(s[e], a.w, x[3]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) *reinterpret_cast<float4*>(parts + (group * DKP + row(e)) * kCols + c0) = s[e];
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kGroups; ++g) add(sum, 1.f, *reinterpret_cast<const float4*>(parts + g * DKP * kCols + mine));
    *out = sum;
    *reinterpret_cast<float4*>(X + mine) = sum;
  }
}

// The blocks of the second half of the grid, if there is one, go backward.
template <int DKP>
__global__ void __launch_bounds__(JoinLayout<DKP>::kThreads) join_kernel(const __grid_constant__ Params p, unsigned half) {
  if (blockIdx.x < half)
    join<DKP, false>(p, blockIdx.x);
  else
    join<DKP, true>(p, blockIdx.x - half);
}

template <int DKP>
cudaError_t run_join(const Params& p, cudaStream_t s) {
  constexpr int smem = JoinLayout<DKP>::kBytes;
  cudaError_t e = allow_smem<join_kernel<DKP>>(smem);
  if (e != cudaSuccess) return e;
  const double cells = (double)p.nsegs * p.hv * DKP * DKP;
  LaunchTimer t("delta_join_kernel", s, 4.0 * cells, 2.0 * cells * p.dv);
  const unsigned half = (unsigned)p.nseq * p.hv * ((p.dv + kCols - 1) / kCols);
  join_kernel<DKP><<<p.backward ? 2 * half : half, JoinLayout<DKP>::kThreads, smem, s>>>(p, half);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_join(const Params& p, cudaStream_t s) {
  if (p.offsets == nullptr && p.nsegs <= 2 * p.nseq) return cudaSuccess;   // nothing between first and last
  return p.dk <= 64 ? run_join<64>(p, s) : run_join<128>(p, s);
}

}  // namespace delta
}  // namespace qrb
