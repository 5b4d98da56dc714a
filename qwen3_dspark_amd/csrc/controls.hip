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
// row change by more than the mask, so the kernel is a copy of the logits with
// bit sets that say where to look closer.
#include <cfloat>
#include <cstring>

#include "common.h"

namespace dspark {

constexpr int LC_CHUNK = 4096;                   // tokens per workgroup
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

constexpr int LC_ROWS = 8;                       // rows of a request between two barriers
constexpr int LC_FLIGHT = 4;                     // 16-byte loads of a thread in flight

// What of a request falls on the CH tokens from v0 on, gathered once per workgroup:
// occurrences in the answer (bit 31: in the prompt), biases, and the proposed
// tokens, which the rows see one after the other.
template <int CH>
struct ControlTables {
  uint32_t seen[CH];
  uint16_t bias[CH];                             // 1 + the request's entry, or 0
  uint32_t touched[CH / 32];                     // any of the above, or proposed
  uint32_t proposed[CH / 32];
  int32_t order[LC_PROPOSED + 1];                // the proposed tokens
  uint32_t allowed[LC_ROWS][CH / 32];            // of the rows at hand
  int32_t any[LC_ROWS];
};

template <int CH>
__device__ __forceinline__ void mark(ControlTables<CH>& t, int at) { atomicOr(&t.touched[at >> 5], 1u << (at & 31)); }

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
    if (i < prompt) atomicOr(&t.seen[at], 0x80000000u);
    else atomicAdd(&t.seen[at], 1u);
    mark(t, (int)at);
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

// The COUNT bits of a set from bit `at` on; no word is read that holds none of them.
template <int COUNT>
__device__ __forceinline__ uint32_t bits_from(const uint32_t* words, int at) {
  const int low = at & 31;
  uint32_t x = words[at >> 5] >> low;
  if (low + COUNT > 32) x |= words[(at >> 5) + 1] << (32 - low);
  return x & ((1u << COUNT) - 1u);
}

// Workgroup (chunk of CH tokens, request): the rows of the request.
//
// Bound by memory for full batches; by the chain of dependent reads for small ones: the layout,
// the text, the logits.  The first logits are therefore loaded ahead of the text, the
// rows' mask words are staged together, and a thread keeps LC_FLIGHT loads in flight,
// over as many rows as it takes.
template <int IN, int OUT, int CH, int T, bool MASK>
__global__ __launch_bounds__(T) void logit_controls_kernel(ControlArgs a) {
  typedef typename LogitType<IN>::type In;
  typedef typename LogitType<OUT>::type Out;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  constexpr int VEC = 16 / (int)sizeof(In);      // values per 16-byte load
  constexpr int GROUPS = CH / VEC;               // per row, at most
  constexpr uint32_t ALL = (1u << VEC) - 1u;
  constexpr float MOST = OUT == 0 ? 0x1.fep127f : FLT_MAX;
  __shared__ __attribute__((aligned(16))) ControlTables<CH> t;
  const int r = blockIdx.y;
  const int v0 = blockIdx.x * CH;
  const int n = min(CH, a.vocab - v0);
  const int tid = threadIdx.x;
  const int32_t* layout = a.layout ? a.layout : a.here;
  const int row0 = layout[r], rows = layout[r + 1] - row0;
  if (rows <= 0) return;
  const int32_t* text = layout + a.n_req + 1;
  const int held = text[a.n_req + r], prompt = text[2 * a.n_req + r];
  const int n_prop = min(rows - 1, LC_PROPOSED);
  const bool in_place = a.logits == a.out;

  auto in_row = [&](int j) { return static_cast<const In*>(a.logits) + (row0 + j) * a.row_stride + v0; };
  auto out_row = [&](int j) { return static_cast<Out*>(a.out) + (row0 + j) * a.out_stride + v0; };
  // 16-byte groups of a row from its first aligned value on; values before and behind
  // them one by one, and all of them where the output's groups are not aligned with these.
  auto lead_of = [&](int j) {
    const int lead = (int)((16 - ((uintptr_t)in_row(j) & 15)) & 15) / (int)sizeof(In);
    return ((uintptr_t)(out_row(j) + lead) & 15) == 0 ? min(lead, n) : n;
  };
  // The mask words of rows j0 .. j0 + LC_ROWS - 1.
  auto stage_masks = [&](int j0) {
    const int last = (n - 1) >> 5, bits = n - 32 * last;
    if (tid < LC_ROWS) t.any[tid] = 0;
    __syncthreads();
    for (int i = tid; i < LC_ROWS * (CH / 32); i += T) {
      const int j = i / (CH / 32), w = i % (CH / 32);
      if (j0 + j >= rows || w > last) continue;
      uint32_t x = a.allowed[(row0 + j0 + j) * a.allowed_stride + (v0 >> 5) + w];
      if (w == last && bits < 32) x &= (1u << bits) - 1u;
      t.allowed[j][w] = x;
      if (x) t.any[j] = 1;
    }
  };
  struct Group {
    u32x4 raw;
    uint32_t keep;
    int j, at;                                   // row behind j0; at < 0: none
  };
  // Group number i of the rows at hand, its logits on their way unless all are masked.
  auto fetch = [&](int j0, int count, int i, Group& s) {
    s.j = i / GROUPS;
    s.at = -1;
    if (s.j >= count) return;
    const int at = lead_of(j0 + s.j) + VEC * (i % GROUPS);
    if (at + VEC > n) return;
    s.at = at;
    s.keep = MASK ? bits_from<VEC>(t.allowed[s.j], at) : ALL;
    if (s.keep) s.raw = *reinterpret_cast<const u32x4*>(in_row(j0 + s.j) + at);
  };
  Group ready[LC_FLIGHT];
  auto fetch_all = [&](int j0, int count, int i) {
    #pragma unroll
    for (int u = 0; u < LC_FLIGHT; ++u) fetch(j0, count, i + T * u, ready[u]);
  };

  if (MASK) stage_masks(0);
  {
    u32x4* zero = reinterpret_cast<u32x4*>(&t);          // seen, bias, touched, proposed
    for (int i = tid; i < (CH + CH / 2 + CH / 16) / 4; i += T) zero[i] = u32x4{0u, 0u, 0u, 0u};
  }
  __syncthreads();
  fetch_all(0, min(rows, LC_ROWS), tid);
  const int64_t first = (int64_t)text[r] * a.history_stride;
  if (a.wide) count_history<CH, T>(t, static_cast<const int64_t*>(a.history) + first, held, prompt, v0, n);
  else count_history<CH, T>(t, static_cast<const int32_t*>(a.history) + first, held, prompt, v0, n);
  const int bias0 = a.bias_start[r], bias1 = a.bias_start[r + 1];
  for (int i = bias0 + tid; i < bias1; i += T) {
    const int at = a.bias_token[i] - v0;
    if (at >= 0 && at < n) {
      t.bias[at] = (uint16_t)(1 + i - bias0);
      mark(t, at);
    }
  }
  if (tid < n_prop) {
    const int64_t tok = a.tokens[row0 - r + tid];
    t.order[tid] = tok >= 0 && tok < a.vocab ? (int32_t)tok : -1;
    const int64_t at = tok - v0;
    if (at >= 0 && at < n) {
      atomicOr(&t.proposed[at >> 5], 1u << (at & 31));
      mark(t, (int)at);
    }
  }
  __syncthreads();
  const double rho = a.penalties[r], inv_rho = 1.0 / rho, alpha_p = a.penalties[a.n_req + r], alpha_f = a.penalties[2 * a.n_req + r];

  auto control = [&](float x, int at, int j) {
    uint32_t seen = t.seen[at];
    if (t.proposed[at >> 5] >> (at & 31) & 1u)
      for (int i = 0; i < min(j, LC_PROPOSED); ++i) seen += t.order[i] == v0 + at ? 1u : 0u;
    const uint32_t c = seen & 0x7fffffffu;
    double y = (double)x;
    if (seen) y = y * (y > 0.0 ? inv_rho : rho);      // off by 2^-52 before the rounding to 24 bits
    if (c) y -= (double)c * alpha_f + alpha_p;
    if (t.bias[at]) y += a.bias_value[bias0 + t.bias[at] - 1];
    // a finite logit stays finite
    if (fabsf(x) <= FLT_MAX) y = fmin(fmax(y, -(double)MOST), (double)MOST);
    return (float)y;
  };

  for (int j0 = 0; j0 < rows; j0 += LC_ROWS) {
    const int count = min(rows - j0, LC_ROWS);
    if (j0) {
      __syncthreads();                           // the rows before are done with their masks
      if (MASK) stage_masks(j0);
      __syncthreads();
    }
    // A row that allows nothing at all is -inf throughout, so that no law of it passes
    // for one; its other chunks are looked at only where this one allows nothing.
    uint32_t empty = 0;
    if (MASK) {
      for (int j = 0; j < count; ++j) {
        if (t.any[j]) continue;
        const uint32_t* words = a.allowed + (row0 + j0 + j) * a.allowed_stride;
        const int last = (a.vocab - 1) >> 5, bits = a.vocab - 32 * last;
        uint32_t hit = 0;
        for (int i = tid; i <= last; i += T) hit |= i == last && bits < 32 ? words[i] & ((1u << bits) - 1u) : words[i];
        if (!__syncthreads_or(hit != 0u)) empty |= 1u << j;
      }
    }
    auto finish = [&](const Group& s) {
      if (s.at < 0) return;
      const int j = j0 + s.j;
      const uint32_t look = bits_from<VEC>(t.touched, s.at) & s.keep;
      if (in_place && s.keep == ALL && !look) return;
      const float fill = empty >> s.j & 1u ? -INFINITY : a.fill;
      float x[VEC];
      #pragma unroll
      for (int u = 0; u < VEC; ++u) {
        const uint32_t w = s.raw[IN == 1 ? u & 3 : (u >> 1) & 3];
        x[u] = __builtin_bit_cast(float, IN == 1 ? w : u & 1 ? w & 0xffff0000u : w << 16);
      }
      // as many turns as the lane with the most such values has, mostly one
      for (uint32_t left = look; left; left &= left - 1u) {
        const int at = __builtin_ctz(left);
        float y = x[0];
        #pragma unroll
        for (int u = 1; u < VEC; ++u) y = at == u ? x[u] : y;
        y = control(y, s.at + at, j);
        #pragma unroll
        for (int u = 0; u < VEC; ++u) x[u] = at == u ? y : x[u];
      }
      #pragma unroll
      for (int u = 0; u < VEC; ++u) x[u] = s.keep >> u & 1u ? x[u] : fill;
      Out* to = out_row(j) + s.at;
      if (OUT == 0) {
        bf16x8 v;
        #pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = (bf16)x[u % VEC];
        __builtin_nontemporal_store(v, reinterpret_cast<bf16x8*>(to));
      } else {
        #pragma unroll
        for (int q = 0; q < VEC / 4; ++q)
          __builtin_nontemporal_store(f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]}, reinterpret_cast<f32x4*>(to + 4 * q));
      }
    };
    for (int i = tid; i < count * GROUPS; i += T * LC_FLIGHT) {
      if (j0 || i != tid) fetch_all(j0, count, i);
      #pragma unroll
      for (int u = 0; u < LC_FLIGHT; ++u) finish(ready[u]);
    }
    auto single = [&](int j, int at) {
      const bool keep = !MASK || (t.allowed[j][at >> 5] >> (at & 31) & 1u);
      float x = (float)in_row(j0 + j)[at];
      if (t.touched[at >> 5] >> (at & 31) & 1u) x = control(x, at, j0 + j);
      out_row(j0 + j)[at] = (Out)(keep ? x : empty >> j & 1u ? -INFINITY : a.fill);
    };
    for (int i = tid; i < count * 2 * VEC; i += T) {       // at most VEC - 1 on either side
      const int j = i / (2 * VEC), e = i % (2 * VEC);
      const int lead = lead_of(j0 + j);
      if (e < VEC) {
        if (e < lead && lead < VEC) single(j, e);
      } else if (lead < VEC) {
        const int at = lead + (n - lead) / VEC * VEC + e - VEC;
        if (at < n) single(j, at);
      }
    }
    for (int j = 0; j < count; ++j)
      if (lead_of(j0 + j) >= VEC)
        for (int at = tid; at < n; at += T) single(j, at);
  }
}

}  // namespace dspark

using namespace dspark;

namespace {

// Up to so many workgroups (two per CU) take 512 threads, which shorten the chain of
// each, and more of them 256, of which more fit a CU.  512 / 256 threads, us a launch: one row of
// 151,936 4.7 / 5.3, 16 requests of up to 6 rows of 32,003 12.1 / 15.9; 64 requests of 8 rows of
// 151,936 79.7 / 73.7, 32 FP32 rows over texts of up to 30,000 27.0 / 24.8.
constexpr int LC_FEW = 512;

template <int IN, int OUT>
int launch_controls(const ControlArgs& a, hipStream_t s) {
  constexpr int CH = LC_CHUNK;
  const dim3 grid((unsigned)((a.vocab + CH - 1) / CH), (unsigned)a.n_req);
  if ((int64_t)grid.x * grid.y <= LC_FEW) {
    if (a.allowed) hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, 512, true>), grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, 512, false>), grid, dim3(512), 0, s, a);
  } else {
    if (a.allowed) hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, 256, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, 256, false>), grid, dim3(256), 0, s, a);
  }
  return launch_status("logit_controls_kernel");
}

}  // namespace

extern "C" int dspark_logit_controls(const void* logits, int dtype, int64_t row_stride, int vocab,
                                     const int32_t* layout, int host_layout, int n_req, const void* history,
                                     int history_bytes, int64_t history_stride, const int64_t* tokens,
                                     const double* penalties, const int32_t* bias_start, const int32_t* bias_token,
                                     const double* bias_value, const int32_t* allowed, int64_t allowed_stride, float fill,
                                     void* out, int out_dtype, int64_t out_stride, void* stream) {
  clear_error();
  DSPARK_REQUIRE(logits && layout && history && penalties && bias_start && out, "null pointer argument");
  DSPARK_REQUIRE(n_req >= 1 && n_req <= 65535, "n_req must be in [1, 65535] (got %d)", n_req);
  DSPARK_REQUIRE(vocab >= 1 && row_stride >= vocab && out_stride >= vocab, "need vocab >= 1 and row strides of at least vocab");
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
  if (dtype == 1) return launch_controls<1, 1>(a, s);
  return out_dtype == 1 ? launch_controls<0, 1>(a, s) : launch_controls<0, 0>(a, s);
}
