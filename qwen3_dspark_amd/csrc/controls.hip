// Penalties, biases and token masks on logits, for gfx950: what stands between
// the LM head and the sampling law when requests bring sampling rules of their own.
//
//   y = x
//   y = y > 0 ? y / rho : y rho        if v occurs in the request's text
//   y = y - c alpha_f - [c > 0] alpha_p   c: occurrences of v in its answer
//   y = y + b_v                        the request's bias of v
//   y = fill                           if the row's mask does not allow v
//
// The text of row j of a request is its history (a prompt, then an answer) and
// the j proposed tokens before the row, which count as answer.  Few values of a
// row change by more than the mask, so the kernel is a copy of the logits under the
// mask, and then a second look at the values that the text touches.
#include <cfloat>
#include <cstring>

#include "common.h"

namespace dspark {

constexpr int LC_PROPOSED = 255;                 // proposed tokens per request

// The batch's layout: cu_rows [n_req + 1], then text [3][n_req] (history row, tokens held,
// of which prompt), in the kernel's arguments for as many requests, else in memory: an
// upload costs a call of one row as much as the kernel takes (27 -> 15 us a call).
constexpr int LC_HERE = 128;

struct ControlArgs {
  const void* logits;
  void* out;
  int64_t row_stride, out_stride;                // elements
  const int32_t* layout;                         // null: `here`
  const void* history;                           // int32 or int64 [.., history_stride]
  int64_t history_stride;
  const int64_t* tokens;                         // proposed, request-major
  const double* penalties;                       // [3][n_req]: rho, alpha_p, alpha_f
  const int32_t* bias_start;                     // [n_req + 1]
  const int32_t* bias_token;
  const double* bias_value;
  const uint32_t* allowed;                       // optional [rows][allowed_stride] words, bit v % 32 of word v / 32
  int64_t allowed_stride;
  float fill;
  int n_req, vocab, wide;                        // wide: history is int64
  int32_t here[4 * LC_HERE + 1];
};

template <int DT>
struct LogitType;
template <>
struct LogitType<0> {
  typedef bf16 type;
};
template <>
struct LogitType<1> {
  typedef float type;
};

constexpr int LC_FLIGHT = 4;                     // 16-byte loads of a thread in flight

// What of a request's text and biases falls on the CH tokens from v0 on, gathered once
// per workgroup: per token the occurrences in the answer and the flags below, and
// the proposed tokens, which the rows see one after the other.
constexpr uint32_t IN_PROMPT = 1u << 31, PROPOSED = 1u << 30, BIASED = 1u << 29, COUNT = BIASED - 1u;

template <int CH>
struct ControlTables {
  uint32_t seen[CH];
  uint16_t bias[CH];                             // the request's entry, where BIASED
  uint16_t list[CH];                             // the tokens with any of these, in any order
  int32_t order[LC_PROPOSED + 1];                // the proposed tokens
  uint8_t any[LC_PROPOSED + 1];                  // rows of which the chunk allows a token
  int32_t count;                                 // tokens in the list
};

// Occurrences of the chunk's tokens in a text, 16 bytes of it per load where its rows allow it.
template <int CH, int T, class Token>
__device__ __forceinline__ void count_history(ControlTables<CH>& t, const Token* text, int held, int prompt, int v0, int n) {
  constexpr int BATCH = 8;
  constexpr int PER = 16 / (int)sizeof(Token);
  typedef Token Pack __attribute__((ext_vector_type(PER)));
  auto count = [&](Token token, int i) {
    // other tokens, and numbers that are none, pass
    const uint32_t at = (uint32_t)token - (uint32_t)v0;
    if (at >= (uint32_t)n || (sizeof(Token) == 8 && (uint64_t)token >> 32)) return;
    if (i < prompt) atomicOr(&t.seen[at], IN_PROMPT);
    else atomicAdd(&t.seen[at], 1u);
  };
  const int packs = ((uintptr_t)text & 15) == 0 ? held / PER : 0;
  for (int p0 = threadIdx.x; p0 < packs; p0 += T * BATCH) {
    Pack pack[BATCH];
    #pragma unroll
    for (int u = 0; u < BATCH; ++u) pack[u] = reinterpret_cast<const Pack*>(text)[min(p0 + T * u, packs - 1)];
    #pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (p0 + T * u < packs) {
        #pragma unroll
        for (int e = 0; e < PER; ++e) count(pack[u][e], PER * (p0 + T * u) + e);
      }
  }
  for (int i0 = PER * packs + threadIdx.x; i0 < held; i0 += T * BATCH) {
    Token token[BATCH];
    #pragma unroll
    for (int u = 0; u < BATCH; ++u) token[u] = text[min(i0 + T * u, held - 1)];
    #pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (i0 + T * u < held) count(token[u], i0 + T * u);
  }
}

// The N (<= 8) bits of a mask row from bit `at` on; no byte is read that holds none of them.
template <int N>
__device__ __forceinline__ uint32_t bits_from(const uint32_t* words, int at) {
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(words);
  uint32_t x = bytes[at >> 3];
  if ((at & 7) + N > 8) x |= (uint32_t)bytes[(at >> 3) + 1] << 8;
  return x >> (at & 7) & ((1u << N) - 1u);
}

// Workgroup (chunk of CH tokens, request): the rows of the request.
//
// First the copy under the mask, 16 bytes a load, LC_FLIGHT of them in flight, values
// that the mask forbids unread; then the text is counted, and each (touched token, row)
// that is allowed is computed by a thread of its own and written over the copy.
// With the look at the text inside the copy, every wave's turn was held up by the one or
// two lanes that a text of a thousand tokens touches (64 requests x 8 rows x 151,936 under
// masks: 218 vector instructions per 16 bytes and lane, now 160; 105 us a call, now 76,
// 4.2 TB/s; a plain copy of the rows 60).
//
// Bound by memory for full batches; by the chain of dependent reads for small ones (one
// row of 151,936 5.4 us).
template <int IN, int OUT, int CH, int T, bool MASK>
__global__ __launch_bounds__(T) void logit_controls_kernel(ControlArgs a) {
  typedef typename LogitType<IN>::type In;
  typedef typename LogitType<OUT>::type Out;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  constexpr int VEC = 16 / (int)sizeof(In);      // values per 16-byte load
  constexpr int PER = VEC / 4;                   // values per word of it
  constexpr int GROUPS = CH / VEC;               // per row, at most
  constexpr float MOST = OUT == 0 ? 0x1.fep127f : FLT_MAX;
  __shared__ __attribute__((aligned(16))) ControlTables<CH> t;
  const int r = blockIdx.y;
  const int v0 = blockIdx.x * CH;
  const int n = min(CH, a.vocab - v0);
  const int tid = threadIdx.x;
  auto layout = [&](int i) { return a.layout ? a.layout[i] : a.here[i]; };
  const int row0 = layout(r), rows = min(layout(r + 1) - row0, LC_PROPOSED + 1);
  if (rows <= 0) return;
  const bool in_place = a.logits == a.out;
  auto in_row = [&](int j) { return static_cast<const In*>(a.logits) + (row0 + j) * a.row_stride + v0; };
  auto out_row = [&](int j) { return static_cast<Out*>(a.out) + (row0 + j) * a.out_stride + v0; };
  auto mask_row = [&](int j) { return a.allowed + (row0 + j) * a.allowed_stride + (v0 >> 5); };
  auto allows = [&](int j, int at) { return !MASK || (mask_row(j)[at >> 5] >> (at & 31) & 1u); };
  // 16-byte groups of a row from its first aligned value on; values before and behind
  // them one by one, and all of them where the output's groups are not aligned with these.
  auto lead_of = [&](int j) {
    const int lead = (int)((16 - ((uintptr_t)in_row(j) & 15)) & 15) / (int)sizeof(In);
    return ((uintptr_t)(out_row(j) + lead) & 15) == 0 ? min(lead, n) : n;
  };

  {
    u32x4* zero = reinterpret_cast<u32x4*>(&t);          // seen
    for (int i = tid; i < CH / 4; i += T) zero[i] = u32x4{0u, 0u, 0u, 0u};
    for (int i = tid; i <= LC_PROPOSED; i += T) t.any[i] = MASK ? 0 : 1;
    if (tid == 0) t.count = 0;
  }
  __syncthreads();

  // The copy.  The 64 groups of a wave are of one row, whose addresses are scalar.
  static_assert(GROUPS % WAVE == 0, "a wave's groups are of one row");
  // In a register: a choice between a logit and the argument would become one of addresses,
  // for which all arguments would be copied to scratch memory.
  const uint32_t fill_bits = (uint32_t)__builtin_amdgcn_readfirstlane((int)__builtin_bit_cast(uint32_t, a.fill));
  const float fill = __builtin_bit_cast(float, fill_bits);
  const uint32_t fill_word = OUT == 1 ? fill_bits : __builtin_bit_cast(uint16_t, (bf16)fill) * 0x10001u;
  for (int i0 = tid; i0 < rows * GROUPS; i0 += T * LC_FLIGHT) {
    u32x4 raw[LC_FLIGHT];
    uint32_t keep[LC_FLIGHT];
    int at[LC_FLIGHT];                           // first value of the group, -1: none
    #pragma unroll
    for (int u = 0; u < LC_FLIGHT; ++u) {
      const int i = i0 + T * u, j = __builtin_amdgcn_readfirstlane(i) / GROUPS;
      at[u] = -1;
      if (j >= rows) continue;
      const int first = lead_of(j) + VEC * (i % GROUPS);
      if (first + VEC <= n) at[u] = first;
      if (at[u] >= 0) keep[u] = MASK ? bits_from<VEC>(mask_row(j), first) : (1u << VEC) - 1u;
    }
    #pragma unroll
    for (int u = 0; u < LC_FLIGHT; ++u) {
      const int j = __builtin_amdgcn_readfirstlane(i0 + T * u) / GROUPS;
      raw[u] = u32x4{0u, 0u, 0u, 0u};
      if (at[u] >= 0 && keep[u]) raw[u] = *reinterpret_cast<const u32x4*>(in_row(j) + at[u]);
    }
    #pragma unroll
    for (int u = 0; u < LC_FLIGHT; ++u) {
      const int j = __builtin_amdgcn_readfirstlane(i0 + T * u) / GROUPS;
      if (at[u] < 0) continue;
      if (MASK && keep[u]) t.any[j] = 1;
      if (in_place && keep[u] == (1u << VEC) - 1u) continue;
      Out* to = out_row(j) + at[u];
      if constexpr (IN == OUT) {
        if (MASK) {
          #pragma unroll
          for (int d = 0; d < 4; ++d) {
            const uint32_t first = 0u - (keep[u] >> (PER * d) & 1u), last = 0u - (keep[u] >> (PER * d + PER - 1) & 1u);
            const uint32_t some = (first & 0xffffu) | (last & 0xffff0000u);
            raw[u][d] = (raw[u][d] & some) | (fill_word & ~some);
          }
        }
        __builtin_nontemporal_store(raw[u], reinterpret_cast<u32x4*>(to));
      } else {
        #pragma unroll
        for (int q = 0; q < 2; ++q) {
          f32x4 x;
          #pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = raw[u][2 * q + (e >> 1)];
            x[e] = __builtin_bit_cast(float, e & 1 ? w & 0xffff0000u : w << 16);
            if (MASK && !(keep[u] >> (4 * q + e) & 1u)) x[e] = fill;
          }
          __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(to + 4 * q));
        }
      }
    }
  }
  auto single = [&](int j, int at) {
    const bool keep = allows(j, at);
    if (MASK && keep) t.any[j] = 1;
    out_row(j)[at] = keep ? (Out)(float)in_row(j)[at] : (Out)fill;
  };
  for (int i = tid; i < rows * 2 * VEC; i += T) {            // at most VEC - 1 on either side
    const int j = i / (2 * VEC), e = i % (2 * VEC);
    const int lead = lead_of(j);
    if (lead >= VEC) continue;
    const int at = e < VEC ? e : lead + (n - lead) / VEC * VEC + e - VEC;
    if (e < VEC ? e < min(lead, n) : at < n) single(j, at);
  }
  for (int j = 0; j < rows; ++j)
    if (lead_of(j) >= VEC)
      for (int at = tid; at < n; at += T) single(j, at);

  // The text.
  const int64_t first = (int64_t)layout(a.n_req + 1 + r) * a.history_stride;
  const int held = layout(2 * a.n_req + 1 + r), prompt = layout(3 * a.n_req + 1 + r);
  if (a.wide) count_history<CH, T>(t, static_cast<const int64_t*>(a.history) + first, held, prompt, v0, n);
  else count_history<CH, T>(t, static_cast<const int32_t*>(a.history) + first, held, prompt, v0, n);
  const int bias0 = a.bias_start[r], bias1 = a.bias_start[r + 1];
  for (int i = bias0 + tid; i < bias1; i += T) {
    const int at = a.bias_token[i] - v0;
    if (at >= 0 && at < n) {
      t.bias[at] = (uint16_t)(i - bias0);
      atomicOr(&t.seen[at], BIASED);
    }
  }
  for (int i = tid; i < rows - 1; i += T) {
    const int64_t token = a.tokens[row0 - r + i];
    const int64_t at = token - v0;
    t.order[i] = at >= 0 && at < n ? (int32_t)at : -1;
    if (at >= 0 && at < n) atomicOr(&t.seen[at], PROPOSED);
  }
  const double rho = a.penalties[r], inv_rho = 1.0 / rho, alpha_p = a.penalties[a.n_req + r], alpha_f = a.penalties[2 * a.n_req + r];
  __syncthreads();
  {
    const int lane = tid & 63;
    uint64_t hit[CH / T];
    int mine = 0;                                // of the wave
    #pragma unroll
    for (int k = 0; k < CH / T; ++k) {
      hit[k] = __builtin_amdgcn_ballot_w64(t.seen[k * T + tid] != 0u);
      mine += __builtin_popcountll(hit[k]);
    }
    int at = 0;
    if (lane == 0 && mine) at = atomicAdd(&t.count, mine);
    at = __builtin_amdgcn_readfirstlane(at);
    #pragma unroll
    for (int k = 0; k < CH / T; ++k) {
      if (hit[k] >> lane & 1u) t.list[at + __builtin_popcountll(hit[k] & ((1ull << lane) - 1ull))] = (uint16_t)(k * T + tid);
      at += __builtin_popcountll(hit[k]);
    }
  }
  __syncthreads();                               // the list, and the copy that is now written over

  // A pair a turn: four of them with their loads in flight took 5 % more where texts are
  // short, and 8 % less where a chunk is all touched (64 requests of 13 rows of 5,000).
  const int pairs = t.count * rows;
  for (int i = tid; i < pairs; i += T) {
    const int at = t.list[i / rows], j = i % rows;
    if (!allows(j, at)) continue;
    const float x = (float)in_row(j)[at];
    const uint32_t seen = t.seen[at];
    uint32_t c = seen & COUNT;
    if (seen & PROPOSED)
      for (int k = 0; k < j; ++k) c += t.order[k] == at ? 1u : 0u;
    double y = (double)x;
    if (c || seen & IN_PROMPT) y *= y > 0.0 ? inv_rho : rho;      // off by 2^-52 before the rounding to 24 bits
    if (c) y -= (double)c * alpha_f + alpha_p;
    if (seen & BIASED) y += a.bias_value[bias0 + t.bias[at]];
    // a finite logit stays finite
    if (fabsf(x) <= FLT_MAX) y = fmin(fmax(y, -(double)MOST), (double)MOST);
    out_row(j)[at] = (Out)(float)y;
  }

  // A row that allows nothing at all is -inf throughout, so that no law of it passes for
  // one: its other chunks are looked at, a wave a row, only where this one allows nothing.
  if (MASK) {
    for (int j = tid >> 6; j < rows; j += T / WAVE) {
      if (t.any[j]) continue;                    // uniform in the wave
      const uint32_t* words = a.allowed + (row0 + j) * a.allowed_stride;
      const int last = (a.vocab - 1) >> 5, bits = a.vocab - 32 * last;
      uint64_t hit = 0;
      for (int w0 = 0; w0 <= last && !hit; w0 += 4 * WAVE) {
        uint32_t x = 0;
        #pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int w = w0 + WAVE * u + (tid & 63);
          if (w <= last) x |= w == last && bits < 32 ? words[w] & ((1u << bits) - 1u) : words[w];
        }
        hit = __builtin_amdgcn_ballot_w64(x != 0u);
      }
      if (!hit)
        for (int at = tid & 63; at < n; at += WAVE) out_row(j)[at] = (Out)-INFINITY;
    }
  }
}

}  // namespace dspark

using namespace dspark;

namespace {

// Chunks of 2,048 tokens: every chunk reads the request's whole text, but small ones keep more
// loads of the copy in flight on a CU (64 requests x 8 rows x 151,936 bf16, texts of up to 2,000:
// 2,048 / 4,096 / 8,192 tokens 85 / 95 / 106 us a call without masks).
//   Up to LC_FEW workgroups (two per CU) take 512 threads, which shorten the chain of
//   each, more of them 256: 512 / 256 threads, us a launch: 16 requests of up to 6 rows of
//   32,003 8.7 / 10.8; the 64 x 8 rows 72 / 64.
//   Where texts are long for the rows, chunks of 8,192 read them less often: 32 FP32 rows of
//   151,936 over texts of up to 30,000 24.3 us, in chunks of 2,048 31.1.  (Both are bound by reading
//   the text through the L1 caches and by the LDS atomics of its most frequent tokens:
//   without a text 8.)
constexpr int LC_FEW = 512;
constexpr int64_t LC_LONG_TEXT = 2048;          // tokens of text per row
constexpr int LONG_CH = 8192, LONG_T = 1024;

template <int IN, int OUT, int CH, int T>
int launch_chunks(const ControlArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.vocab + CH - 1) / CH), (unsigned)a.n_req);
  if (a.allowed) hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, T, true>), grid, dim3(T), 0, s, a);
  else hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, T, false>), grid, dim3(T), 0, s, a);
  return launch_status("logit_controls_kernel");
}

template <int IN, int OUT>
int launch_controls(const ControlArgs& a, int64_t text_tokens, int64_t rows, hipStream_t s) {
  if (text_tokens > LC_LONG_TEXT * rows) return launch_chunks<IN, OUT, LONG_CH, LONG_T>(a, s);
  if ((int64_t)a.n_req * ((a.vocab + 2047) / 2048) <= LC_FEW) return launch_chunks<IN, OUT, 2048, 512>(a, s);
  return launch_chunks<IN, OUT, 2048, 256>(a, s);
}

}  // namespace

extern "C" int dspark_logit_controls(const void* logits, int dtype, int64_t row_stride, int vocab,
                                     const int32_t* layout, int host_layout, int n_req, int64_t rows,
                                     int64_t text_tokens, const void* history, int history_bytes,
                                     int64_t history_stride, const int64_t* tokens,
                                     const double* penalties, const int32_t* bias_start, const int32_t* bias_token,
                                     const double* bias_value, const int32_t* allowed, int64_t allowed_stride, float fill,
                                     void* out, int out_dtype, int64_t out_stride, void* stream) {
  clear_error();
  DSPARK_REQUIRE(logits && layout && history && penalties && bias_start && out, "null pointer argument");
  DSPARK_REQUIRE(n_req >= 1 && n_req <= 65535, "n_req must be in [1, 65535] (got %d)", n_req);
  DSPARK_REQUIRE(rows >= 1 && text_tokens >= 0, "need rows >= 1 and text_tokens >= 0");
  DSPARK_REQUIRE(vocab >= 1 && vocab <= (1 << 30) && row_stride >= vocab && out_stride >= vocab,
                 "need vocab in [1, 2^30] and row strides of at least vocab");
  DSPARK_REQUIRE(dtype == 0 || dtype == 1, "dtype must be 0 (bf16) or 1 (fp32)");
  DSPARK_REQUIRE(out_dtype == 1 || out_dtype == dtype, "out_dtype must be the logits' or 1 (fp32)");
  DSPARK_REQUIRE(history_bytes == 4 || history_bytes == 8, "history must be int32 or int64");
  DSPARK_REQUIRE(history_stride >= 0 && (!allowed || allowed_stride >= (vocab + 31) / 32), "a mask row needs ceil(vocab / 32) words");
  DSPARK_REQUIRE(logits != out || (dtype == out_dtype && row_stride == out_stride), "in place needs one type and row stride");
  DSPARK_REQUIRE(!host_layout || n_req <= LC_HERE, "a layout in host memory is of at most %d requests", LC_HERE);
  ControlArgs a{logits, out, row_stride, out_stride, host_layout ? nullptr : layout, history, history_stride, tokens, penalties, bias_start,
                bias_token, bias_value, reinterpret_cast<const uint32_t*>(allowed), allowed_stride, fill, n_req, vocab,
                history_bytes == 8, {}};
  if (host_layout) std::memcpy(a.here, layout, sizeof(int32_t) * (4 * n_req + 1));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == 1) return launch_controls<1, 1>(a, text_tokens, rows, s);
  return out_dtype == 1 ? launch_controls<0, 1>(a, text_tokens, rows, s) : launch_controls<0, 0>(a, text_tokens, rows, s);
}
