// Low-rank adapters beside the shared q/k/v projection, the part that runs inside
// the projection kernels:
//   C^T[dim][token] += B_a[dim][:] . u[token][:],   u = s_a A_a x, a the token's adapter.
// u comes from the shrinking launch (adapters.hip) as two bf16 numbers per value (the value
// rounded, and the rest rounded), so that it reaches the product to 16 bits: as one
// bf16 number its rounding would be as large as the output's own.
//
// Bound like the projection around it by latency for small batches and by the matrix unit
// for prompts.  With / without adapters, us of the projection's launch: one token of rank 8 8.6 /
// 7.9, 64 requests x 7 tokens of rank 16 over 24 adapters 12.8 / 10.9, 3,714 tokens of rank 32 of 4
// adapters 51.0 / 45.6.
#pragma once
#include "head_gemm.h"

namespace dspark {

struct AdapterArgs {
  const int32_t* token;        // [T] the adapter of each token, or -1
  const bf16* b;               // [adapters][32 heads (q, k, v)][128][rank]
  const bf16* u;               // [3 (q, k, v)][T][2][rank]
  int adapters;
  int rank;                    // 16, 32 or a multiple of 64, the columns behind an adapter's own rank zero
  int tile_tokens;             // tokens per workgroup of the narrow tiles (adapter_tile_tokens)
};

struct ShrinkArgs {
  const bf16* x;               // [T, hidden]
  const bf16* a;               // [adapters][3][rank][hidden]
  const float* scaling;        // [adapters]
  const int32_t* tiles;        // [n_tiles][4]: first token, tokens, adapter, 0
  bf16* u;                     // [3][T][2][rank]
  int tokens, hidden, adapters, rank, ranks;     // ranks: of which an adapter has its own
};
int launch_adapter_shrink(const ShrinkArgs& s, int n_tiles, int tile_tokens, hipStream_t stream);

// Adds the adapters' part to the accumulators of TT x 32 tokens by 2 x 32 dims of one
// wave (MFMA layout of head_gemm.h: row = dim, column = token).  acc(i, tt): the accumulator
// of dim tile i; rows(i): the weight row of the lane in it; id[tt], u[tt]: the adapter and u
// of the lane's token.  The adapters among the wave's tokens are taken one after the
// other, the next one's weights on their way meanwhile; each column keeps the
// products of its own adapter only, so that no value of another request's
// adapter reaches it, an infinity or NaN neither.
//   RK: 16-wide steps of the rank taken together (the rank is a multiple of 16 RK), which
//   PARTS waves divide among them; a single step they take adapter by adapter.
template <int TT, int RK, int PARTS, class Acc, class Rows>
__device__ __forceinline__ void adapter_expand(Acc acc, const AdapterArgs& ad, int head, const int (&id)[TT],
                                               const bf16* const (&u)[TT], Rows rows, int part) {
  constexpr int OWN = RK >= PARTS ? RK / PARTS : 1;          // steps of this wave per adapter
  static_assert(OWN * PARTS == RK || RK == 1, "the steps divide evenly");
  const int k0 = 8 * ((threadIdx.x & 63) >> 5) + (RK >= PARTS ? 16 * OWN * part : 0);
  for (int block = 0; block < ad.rank; block += 16 * RK) {
    bf16x8 hi[TT][OWN], lo[TT][OWN];
    #pragma unroll
    for (int tt = 0; tt < TT; ++tt)
      #pragma unroll
      for (int o = 0; o < OWN; ++o) {
        hi[tt][o] = ld8(u[tt] + block + k0 + 16 * o);
        lo[tt][o] = ld8(u[tt] + ad.rank + block + k0 + 16 * o);
      }
    bool open[TT];
    #pragma unroll
    for (int tt = 0; tt < TT; ++tt) open[tt] = id[tt] >= 0 && id[tt] < ad.adapters;
    // The next adapter of the wave's tokens, its tokens closed; -1: none.
    auto next = [&]() {
      int cur = -1;
      #pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const uint64_t left = __builtin_amdgcn_ballot_w64(open[tt]);
        if (cur < 0 && left) cur = __builtin_amdgcn_readlane(id[tt], __builtin_ctzll(left));
      }
      #pragma unroll
      for (int tt = 0; tt < TT; ++tt) open[tt] = open[tt] && id[tt] != cur;
      return cur;
    };
    // The same, of the adapters that this wave takes.
    int turn = 0;
    auto mine = [&]() {
      int cur = next();
      if (RK < PARTS)
        for (; cur >= 0 && (turn++ & (PARTS - 1)) != part;) cur = next();
      return cur;
    };
    bf16x8 w[2][OWN];
    auto load = [&](int cur) {
      const bf16* from = ad.b + ((size_t)cur * (HQ + 2 * HKV) + head) * HD * ad.rank + block + k0;
      #pragma unroll
      for (int i = 0; i < 2; ++i)
        #pragma unroll
        for (int o = 0; o < OWN; ++o) w[i][o] = ld8(from + (size_t)rows(i) * ad.rank + 16 * o);
    };
    int cur = mine();
    if (cur >= 0) load(cur);
    while (cur >= 0) {
      bf16x8 here[2][OWN];
      #pragma unroll
      for (int i = 0; i < 2; ++i)
        #pragma unroll
        for (int o = 0; o < OWN; ++o) here[i][o] = w[i][o];
      const int following = mine();
      if (following >= 0) load(following);
      #pragma unroll
      for (int tt = 0; tt < TT; ++tt)
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x16 d = {};
          #pragma unroll
          for (int o = 0; o < OWN; ++o) {
            d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(here[i][o], hi[tt][o], d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(here[i][o], lo[tt][o], d, 0, 0, 0);
          }
          f32x16& c = acc(i, tt);
          #pragma unroll
          for (int e = 0; e < 16; ++e) c[e] += id[tt] == cur ? d[e] : 0.f;
        }
      cur = following;
    }
  }
}

// Ranks that the kernels take (adapters are laid out with zeros up to one).
inline bool adapter_rank(int rank) { return rank == 16 || rank == 32 || (rank >= 64 && rank % 64 == 0 && rank <= 256); }

// Tokens per narrow tile of a batch with adapters: as few as leave one workgroup per CU (8
// tiles of each of 32 heads), since a tile takes its adapters one after the other, while the
// shared weights of its head come from the L2 that all tiles of the head share: 32 tokens
// each with an adapter of rank 64 11.8 us in tiles of 4, in one of 32 24.8.  Above 256 tokens
// the tiles of 64 fill the CUs by themselves.
inline int adapter_tile_tokens(int tokens) { return tokens <= 256 ? (tokens + 7) / 8 : 64; }

}  // namespace dspark
