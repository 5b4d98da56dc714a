// Low-rank adapters of many requests, the shrinking half, for gfx950:
//   u[p][t][:] = s_a A_{a,p} x_t      p = q, k, v; a = the adapter of token t
// stored as two bf16 numbers per value (adapters.h).  The projection kernels add B u.
//
// Work: one workgroup per (16 tokens of one adapter, 16 ranks of one projection);
// its 4 waves divide the hidden columns and add their sums through LDS.
// MFMA 16x16x32: A = 16 adapter rows, B = 16 tokens, both straight from memory
// (a lane's operand is 16 contiguous bytes of a row, and each row is used once here).
#include "adapters.h"

namespace dspark {

constexpr int SH_TOKENS = 16;
constexpr int SH_WAVES = 4;
constexpr int SH_BATCH = 8;                      // 32-column steps of a wave in flight

struct ShrinkArgs {
  const bf16* x;               // [T, hidden]
  const bf16* a;               // [adapters][3][rank][hidden]
  const float* scaling;        // [adapters]
  const int32_t* tiles;        // [n_tiles][4]: first token, tokens (<= 16), adapter, 0
  bf16* u;                     // [3][T][2][rank]
  int tokens, hidden, adapters, rank, ranks;     // ranks: of which an adapter has its own
};

__global__ __launch_bounds__(SH_WAVES * WAVE) void adapter_shrink_kernel(ShrinkArgs s) {
  __shared__ f32x4 sums[SH_WAVES][WAVE];
  const int32_t* tile = s.tiles + 4 * blockIdx.x;
  const int t0 = tile[0], n = tile[1], adapter = tile[2];
  if (t0 < 0 || n < 1 || t0 + n > s.tokens || adapter < 0 || adapter >= s.adapters) return;   // uniform
  const int p = blockIdx.y % 3, r0 = (blockIdx.y / 3) * 16;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int col = lane & 15, grp = lane >> 4;
  const bf16* arow = s.a + (((size_t)adapter * 3 + p) * s.rank + r0 + col) * s.hidden + 8 * grp;
  const bf16* xrow = s.x + (size_t)(t0 + min(col, n - 1)) * s.hidden + 8 * grp;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int steps = s.hidden / (32 * SH_WAVES);        // of this wave: columns 32 (SH_WAVES i + wave) ..
  for (int i0 = 0; i0 < steps; i0 += SH_BATCH) {
    bf16x8 av[SH_BATCH], xv[SH_BATCH];
    #pragma unroll
    for (int b = 0; b < SH_BATCH; ++b) {
      const int c = 32 * (SH_WAVES * min(i0 + b, steps - 1) + wave);
      av[b] = ld8(arow + c);
      xv[b] = ld8(xrow + c);
    }
    #pragma unroll
    for (int b = 0; b < SH_BATCH; ++b)
      if (i0 + b < steps) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[b], xv[b], acc, 0, 0, 0);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
  f32x4 v = sums[0][lane];
  #pragma unroll
  for (int w = 1; w < SH_WAVES; ++w) v += sums[w][lane];
  if (col >= n) return;
  const float scale = s.scaling[adapter];
  bf16x4 hi, lo;
  #pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = r0 + 4 * grp + e < s.ranks ? v[e] * scale : 0.f;
    hi[e] = (bf16)y;
    lo[e] = fabsf((float)hi[e]) <= 3.4e38f ? (bf16)(y - (float)hi[e]) : (bf16)0.f;    // no rest of an infinity
  }
  bf16* out = s.u + ((size_t)p * s.tokens + t0 + col) * 2 * s.rank + r0 + 4 * grp;
  *reinterpret_cast<bf16x4*>(out) = hi;
  *reinterpret_cast<bf16x4*>(out + s.rank) = lo;
}

}  // namespace dspark

using namespace dspark;

extern "C" int dspark_adapter_shrink(const void* x, int tokens, int hidden, const void* a, const float* scaling,
                                     int adapters, int rank, int own_rank, const int32_t* tiles, int n_tiles, void* u,
                                     void* stream) {
  clear_error();
  DSPARK_REQUIRE(x && a && scaling && tiles && u, "null pointer argument");
  DSPARK_REQUIRE(tokens >= 1 && hidden >= HG_COLS && hidden % HG_COLS == 0, "need tokens >= 1 and hidden a multiple of %d",
                 HG_COLS);
  DSPARK_REQUIRE(adapters >= 1 && rank >= 16 && rank % 16 == 0 && rank <= 256 && own_rank >= 1 && own_rank <= rank,
                 "need adapters >= 1, rank a multiple of 16 up to 256 and own_rank in [1, rank]");
  DSPARK_REQUIRE(n_tiles >= 1, "n_tiles must be >= 1");
  DSPARK_REQUIRE((((uintptr_t)x | (uintptr_t)a | (uintptr_t)u) & 15) == 0, "tensors must be 16-byte aligned");
  ShrinkArgs s{static_cast<const bf16*>(x), static_cast<const bf16*>(a), scaling, tiles, static_cast<bf16*>(u), tokens,
               hidden, adapters, rank, own_rank};
  hipLaunchKernelGGL(adapter_shrink_kernel, dim3((unsigned)n_tiles, 3 * rank / 16), dim3(SH_WAVES * WAVE), 0,
                     static_cast<hipStream_t>(stream), s);
  return launch_status("adapter_shrink_kernel");
}
