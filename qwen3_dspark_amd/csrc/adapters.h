// Low-rank adapters beside the shared q/k/v projection, the part that runs inside
// the projection kernels:
//   C^T[dim][token] += B_a[dim][:] . u[token][:],   u = s_a A_a x, a the token's adapter.
// u comes from dspark_adapter_shrink as two bf16 numbers per value (the value
// rounded, and the rest rounded), so that it reaches the product to 16 bits: as one
// bf16 number its rounding would be as large as the output's own.
#pragma once
#include "head_gemm.h"

namespace dspark {

struct AdapterArgs {
  const int32_t* token;        // [T] the adapter of each token, or -1
  const bf16* b;               // [adapters][32 heads (q, k, v)][128][rank]
  const bf16* u;               // [3 (q, k, v)][T][2][rank]
  int adapters;
  int rank;                    // a multiple of 16, the columns behind an adapter's own rank zero
};

// Adds the adapters' part to the accumulators of TT x 32 tokens by 2 x 32 dims of one
// wave (MFMA layout of head_gemm.h: row = dim, column = token).  rows(i): the
// weight row of the lane in dim tile i; token id[tt] and u[tt] of the lane's column.
// The adapters among the wave's tokens are taken one after the other; each
// column keeps the products of its own adapter only, so that no value of another
// request's adapter reaches it, an infinity or NaN neither.  Of the 16-wide steps
// this wave takes those with number = part modulo `parts`.
template <int TT, class Acc, class Rows>
__device__ __forceinline__ void adapter_expand(Acc&& acc, const AdapterArgs& ad, int head, const int (&id)[TT],
                                               const bf16* const (&u)[TT], Rows rows, int part, int parts) {
  const int lane = threadIdx.x & 63;
  const int hl = lane >> 5;
  bool open[TT];
  #pragma unroll
  for (int tt = 0; tt < TT; ++tt) open[tt] = id[tt] >= 0 && id[tt] < ad.adapters;
  int step = 0;
  for (;;) {
    int cur = -1;
    #pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const uint64_t left = __builtin_amdgcn_ballot_w64(open[tt]);
      if (cur < 0 && left) cur = __builtin_amdgcn_readlane(id[tt], __builtin_ctzll(left));
    }
    if (cur < 0) break;
    const bf16* w = ad.b + ((size_t)cur * (HQ + 2 * HKV) + head) * HD * ad.rank + 8 * hl;
    f32x16 d[2][TT];
    #pragma unroll
    for (int i = 0; i < 2; ++i)
      #pragma unroll
      for (int tt = 0; tt < TT; ++tt) d[i][tt] = f32x16{};
    for (int ks = 0; ks < ad.rank; ks += 16, ++step) {
      if (step % parts != part) continue;
      bf16x8 wa[2];
      #pragma unroll
      for (int i = 0; i < 2; ++i) wa[i] = ld8(w + (size_t)rows(i) * ad.rank + ks);
      #pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const bf16x8 hi = ld8(u[tt] + ks + 8 * hl), lo = ld8(u[tt] + ad.rank + ks + 8 * hl);
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          d[i][tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[i], hi, d[i][tt], 0, 0, 0);
          d[i][tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[i], lo, d[i][tt], 0, 0, 0);
        }
      }
    }
    #pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const bool mine = id[tt] == cur;
      open[tt] = open[tt] && !mine;
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x16& c = acc(i, tt);
        #pragma unroll
        for (int e = 0; e < 16; ++e) c[e] += mine ? d[i][tt][e] : 0.f;
      }
    }
  }
}

}  // namespace dspark
