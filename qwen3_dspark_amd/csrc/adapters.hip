// Low-rank adapters of many requests, the shrinking half, for gfx950:
//   u[p][t][:] = s_a A_{a,p} x_t      p = q, k, v; a = the adapter of token t
// stored as two bf16 numbers per value (adapters.h).  The projection kernels add B u.
//
// Work: one workgroup per (16 tokens of one adapter, 16 ranks) and projection, or per 32
// tokens for all three projections, whose token operands are the same; its waves divide the
// hidden columns and add their sums through LDS.  MFMA 16x16x32: A = 16 adapter rows, B = 16
// tokens, both straight from memory (a lane's operand is 16 contiguous bytes of a row).
// Bound by the one round trip of its loads, all of which are in flight at once, and for
// prompts by the adapter's rows that every tile reads from the L2 again.
#include "adapters.h"

namespace dspark {

// P: projections per workgroup (3, or 1 with blockIdx.z naming it); W: its waves; SH_BATCH: 32-column
// steps of a wave in flight; SUBS: groups of 16 tokens per tile, for all of which an adapter's
// row is read once.
template <int P, int W, int SH_BATCH, int SUBS>
__global__ __launch_bounds__(W * WAVE) void adapter_shrink_kernel(ShrinkArgs s) {
  __shared__ f32x4 sums[W][SUBS][P][WAVE];
  const int32_t* tile = s.tiles + 4 * blockIdx.x;
  const int t0 = tile[0], n = tile[1], adapter = tile[2];
  if (t0 < 0 || n < 1 || n > 16 * SUBS || t0 > s.tokens - n || adapter < 0 || adapter >= s.adapters) return;   // uniform
  const int r0 = blockIdx.y * 16;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int p0 = P == 3 ? 0 : blockIdx.z;
  const bf16* arow = s.a + (((size_t)adapter * 3 + p0) * s.rank + r0 + col) * s.hidden + 8 * grp;
  const size_t next = (size_t)s.rank * s.hidden;                                 // the next projection's rows
  const bf16* xrow[SUBS];
  #pragma unroll
  for (int q = 0; q < SUBS; ++q) xrow[q] = s.x + (size_t)(t0 + min(16 * q + col, n - 1)) * s.hidden + 8 * grp;
  f32x4 acc[SUBS][P] = {};
  const int steps = s.hidden / 32;                       // this wave's: wave, wave + W, ..
  for (int i0 = wave; i0 < steps; i0 += W * SH_BATCH) {
    bf16x8 av[P][SH_BATCH], xv[SUBS][SH_BATCH];
    #pragma unroll
    for (int b = 0; b < SH_BATCH; ++b) {
      const int c = 32 * min(i0 + W * b, steps - 1);
      #pragma unroll
      for (int q = 0; q < SUBS; ++q) xv[q][b] = ld8(xrow[q] + c);
      #pragma unroll
      for (int p = 0; p < P; ++p) av[p][b] = ld8(arow + p * next + c);
    }
    #pragma unroll
    for (int b = 0; b < SH_BATCH; ++b)
      if (i0 + W * b < steps) {
        #pragma unroll
        for (int q = 0; q < SUBS; ++q)
          #pragma unroll
          for (int p = 0; p < P; ++p) acc[q][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[p][b], xv[q][b], acc[q][p], 0, 0, 0);
      }
  }
  #pragma unroll
  for (int q = 0; q < SUBS; ++q)
    #pragma unroll
    for (int p = 0; p < P; ++p) sums[wave][q][p][lane] = acc[q][p];
  __syncthreads();
  const float scale = s.scaling[adapter];
  static_assert(SUBS * P <= W, "a wave per group and projection");
  if (wave >= SUBS * P) return;
  const int q = wave / P, p = wave % P, at = 16 * q + col;
  f32x4 v = sums[0][q][p][lane];
  #pragma unroll
  for (int w = 1; w < W; ++w) v += sums[w][q][p][lane];
  if (at >= n) return;
  bf16x4 hi, lo;
  #pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = r0 + 4 * grp + e < s.ranks ? v[e] * scale : 0.f;
    hi[e] = (bf16)y;
    lo[e] = fabsf((float)hi[e]) <= 3.4e38f ? (bf16)(y - (float)hi[e]) : (bf16)0.f;    // no rest of an infinity
  }
  bf16* out = s.u + ((size_t)(p0 + p) * s.tokens + t0 + at) * 2 * s.rank + r0 + 4 * grp;
  *reinterpret_cast<bf16x4*>(out) = hi;
  *reinterpret_cast<bf16x4*>(out + s.rank) = lo;
}

// Tiles of 16 tokens go to a workgroup per projection, tiles of 32 to one for all three, which
// reads the tokens once and an adapter's rows once for twice as many.  A batch takes the 16s
// up to 256 (16-token tile, 16 ranks) pairs, a workgroup per CU and projection.  16 / 32, us a
// launch: 1,200 tokens of one adapter of rank 16 4.9 / 7.8, 2,048 of rank 16 6.0 / 8.0, 900 of rank 64
// 8.8 / 8.7; 600 of rank 128 10.8 / 9.0, 3,714 of 4 adapters of rank 32 13.7 / 8.2 (all three
// projections of 16 tokens 10.4), 4,000 of 4 of rank 64 24.4 / 12.8.  The loads of small calls fit
// one batch: 8 waves of 4 steps as fast as 4 of 8 or 16 of 2; of large ones 6 or 16 waves
// 9.7 and 8.9 for 8.2.
int launch_adapter_shrink(const ShrinkArgs& s, int n_tiles, int tile_tokens, hipStream_t stream) {
  if (tile_tokens == 16)
    hipLaunchKernelGGL((adapter_shrink_kernel<1, 8, 4, 1>), dim3((unsigned)n_tiles, s.rank / 16, 3), dim3(8 * WAVE), 0, stream, s);
  else
    hipLaunchKernelGGL((adapter_shrink_kernel<3, 8, 4, 2>), dim3((unsigned)n_tiles, s.rank / 16), dim3(8 * WAVE), 0, stream, s);
  return launch_status("adapter_shrink_kernel");
}

}  // namespace dspark
