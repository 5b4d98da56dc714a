// Low-rank adapters of many requests, the shrinking half, for gfx950:
//   u[p][t][:] = s_a A_{a,p} x_t      p = q, k, v; a = the adapter of token t
// stored as two bf16 numbers per value (adapters.h).  The projection kernels add B u.
//
// Work: one workgroup per (16 tokens of one adapter, 16 ranks), all three projections, whose
// token operands are the same; its waves divide the hidden columns and add their sums
// through LDS.  MFMA 16x16x32: A = 16 adapter rows, B = 16 tokens, both straight from
// memory (a lane's operand is 16 contiguous bytes of a row, which is used once here).
// Bound by the one round trip of its loads, all of which are in flight at once.
#include "adapters.h"

namespace dspark {

constexpr int SH_TOKENS = 16;

// P: projections per workgroup (3, or 1 with blockIdx.z naming it); W: its waves; SH_BATCH: 32-column
// steps of a wave in flight.
template <int P, int W, int SH_BATCH>
__global__ __launch_bounds__(W * WAVE) void adapter_shrink_kernel(ShrinkArgs s) {
  __shared__ f32x4 sums[W][P][WAVE];
  const int32_t* tile = s.tiles + 4 * blockIdx.x;
  const int t0 = tile[0], n = tile[1], adapter = tile[2];
  if (t0 < 0 || n < 1 || n > SH_TOKENS || t0 > s.tokens - n || adapter < 0 || adapter >= s.adapters) return;   // uniform
  const int r0 = blockIdx.y * 16;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int p0 = P == 3 ? 0 : blockIdx.z;
  const bf16* arow = s.a + (((size_t)adapter * 3 + p0) * s.rank + r0 + col) * s.hidden + 8 * grp;
  const size_t next = (size_t)s.rank * s.hidden;                                 // the next projection's rows
  const bf16* xrow = s.x + (size_t)(t0 + min(col, n - 1)) * s.hidden + 8 * grp;
  f32x4 acc[P] = {};
  const int steps = s.hidden / 32;                       // this wave's: wave, wave + W, ..
  for (int i0 = wave; i0 < steps; i0 += W * SH_BATCH) {
    bf16x8 av[P][SH_BATCH], xv[SH_BATCH];
    #pragma unroll
    for (int b = 0; b < SH_BATCH; ++b) {
      const int c = 32 * min(i0 + W * b, steps - 1);
      xv[b] = ld8(xrow + c);
      #pragma unroll
      for (int p = 0; p < P; ++p) av[p][b] = ld8(arow + p * next + c);
    }
    #pragma unroll
    for (int b = 0; b < SH_BATCH; ++b)
      if (i0 + W * b < steps) {
        #pragma unroll
        for (int p = 0; p < P; ++p) acc[p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[p][b], xv[b], acc[p], 0, 0, 0);
      }
  }
  #pragma unroll
  for (int p = 0; p < P; ++p) sums[wave][p][lane] = acc[p];
  __syncthreads();
  const float scale = s.scaling[adapter];
  if (wave >= P) return;
  const int p = wave;
  f32x4 v = sums[0][p][lane];
  #pragma unroll
  for (int w = 1; w < W; ++w) v += sums[w][p][lane];
  if (col >= n) return;
  bf16x4 hi, lo;
  #pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = r0 + 4 * grp + e < s.ranks ? v[e] * scale : 0.f;
    hi[e] = (bf16)y;
    lo[e] = fabsf((float)hi[e]) <= 3.4e38f ? (bf16)(y - (float)hi[e]) : (bf16)0.f;    // no rest of an infinity
  }
  bf16* out = s.u + ((size_t)(p0 + p) * s.tokens + t0 + col) * 2 * s.rank + r0 + 4 * grp;
  *reinterpret_cast<bf16x4*>(out) = hi;
  *reinterpret_cast<bf16x4*>(out + s.rank) = lo;
}

// Up to so many (token tile, rank tile) pairs take a workgroup per projection, more of
// them one for all three, which reads the tokens once.  A workgroup per projection /
// for all, us a launch: one token at rank 8 3.4 / 5.1, 64 requests x 7 tokens over 24 adapters of
// rank 16 4.5 / 6.5, 32 tokens each with an adapter of rank 64 5.8 / 7.0, 4,000 tokens of 4
// adapters of rank 32 13.7 / 10.4.  The loads of small calls fit one batch: 8 waves of 4
// steps as fast as 4 of 8 or 16 of 2.
constexpr int SH_FEW = 256;

int launch_adapter_shrink(const ShrinkArgs& s, int n_tiles, hipStream_t stream) {
  if ((int64_t)n_tiles * (s.rank / 16) <= SH_FEW)
    hipLaunchKernelGGL((adapter_shrink_kernel<1, 8, 4>), dim3((unsigned)n_tiles, s.rank / 16, 3), dim3(8 * WAVE), 0, stream, s);
  else
    hipLaunchKernelGGL((adapter_shrink_kernel<3, 8, 2>), dim3((unsigned)n_tiles, s.rank / 16), dim3(8 * WAVE), 0, stream, s);
  return launch_status("adapter_shrink_kernel");
}

}  // namespace dspark
