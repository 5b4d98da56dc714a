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

#include "common.h"

namespace dspark {

constexpr int LC_THREADS = 256;
constexpr int LC_PROPOSED = 255;                 // proposed tokens per request

struct ControlArgs {
  const void* logits;
  void* out;
  int64_t row_stride, out_stride;                // elements
  const int32_t* cu_rows;                        // [n_req + 1]
  const int32_t* text;                           // [3][n_req]: history row, tokens held, of which prompt
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
};

template <int T>
struct LogitType;
template <>
struct LogitType<0> {
  typedef bf16 type;
};
template <>
struct LogitType<1> {
  typedef float type;
};

// What of a request falls on the CH tokens from v0 on, gathered once per workgroup:
// occurrences in the answer (bit 31: in the prompt), biases, and the proposed
// tokens, which the rows see one after the other.
template <int CH>
struct ControlTables {
  uint32_t seen[CH];
  int32_t bias[CH];                              // 1 + the bias's entry, or 0
  uint32_t touched[CH / 32];                 // any of the above, or proposed
  uint32_t proposed[CH / 32];
  int32_t order[LC_PROPOSED + 1];                // the proposed tokens
};

template <int CH>
__device__ __forceinline__ void mark(ControlTables<CH>& t, int at) { atomicOr(&t.touched[at >> 5], 1u << (at & 31)); }

template <int CH, class Token>
__device__ __forceinline__ void count_history(ControlTables<CH>& t, const Token* text, int held, int prompt, int v0, int n) {
  constexpr int BATCH = 8;
  for (int i0 = threadIdx.x; i0 < held; i0 += LC_THREADS * BATCH) {
    int64_t tok[BATCH];
    #pragma unroll
    for (int u = 0; u < BATCH; ++u) tok[u] = (int64_t)text[min(i0 + LC_THREADS * u, held - 1)];
    #pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + LC_THREADS * u;
      const int64_t at = tok[u] - v0;
      if (i < held && at >= 0 && at < n) {       // other tokens, and numbers that are none, pass
        if (i < prompt) atomicOr(&t.seen[at], 0x80000000u);
        else atomicAdd(&t.seen[at], 1u);
        mark(t, (int)at);
      }
    }
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

// Workgroup (chunk of CH tokens, request): the rows of the request, one after the other.
template <int IN, int OUT, int CH, bool MASK>
__global__ __launch_bounds__(LC_THREADS) void logit_controls_kernel(ControlArgs a) {
  typedef typename LogitType<IN>::type In;
  typedef typename LogitType<OUT>::type Out;
  constexpr int VEC = 16 / (int)sizeof(In);      // values per 16-byte load
  constexpr float MOST = OUT == 0 ? 0x1.fep127f : FLT_MAX;
  __shared__ ControlTables<CH> t;
  const int r = blockIdx.y;
  const int v0 = blockIdx.x * CH;
  const int n = min(CH, a.vocab - v0);
  const int tid = threadIdx.x;
  const int row0 = a.cu_rows[r], rows = a.cu_rows[r + 1] - row0;
  if (rows <= 0) return;
  const int n_prop = min(rows - 1, LC_PROPOSED);
  for (int i = tid; i < CH; i += LC_THREADS) {
    t.seen[i] = 0u;
    t.bias[i] = 0;
  }
  for (int i = tid; i < CH / 32; i += LC_THREADS) t.touched[i] = t.proposed[i] = 0u;
  __syncthreads();
  const int held = a.text[a.n_req + r], prompt = a.text[2 * a.n_req + r];
  const int64_t first = (int64_t)a.text[r] * a.history_stride;
  if (a.wide) count_history(t, static_cast<const int64_t*>(a.history) + first, held, prompt, v0, n);
  else count_history(t, static_cast<const int32_t*>(a.history) + first, held, prompt, v0, n);
  for (int i = a.bias_start[r] + tid; i < a.bias_start[r + 1]; i += LC_THREADS) {
    const int at = a.bias_token[i] - v0;
    if (at >= 0 && at < n) {
      t.bias[at] = 1 + i;
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
  const double rho = a.penalties[r], alpha_p = a.penalties[a.n_req + r], alpha_f = a.penalties[2 * a.n_req + r];

  auto control = [&](float x, int at, int j) {
    uint32_t seen = t.seen[at];
    if (t.proposed[at >> 5] >> (at & 31) & 1u)
      for (int i = 0; i < min(j, LC_PROPOSED); ++i) seen += t.order[i] == v0 + at ? 1u : 0u;
    const uint32_t c = seen & 0x7fffffffu;
    double y = (double)x;
    if (seen) y = y > 0.0 ? y / rho : y * rho;
    if (c) y -= (double)c * alpha_f + alpha_p;
    if (t.bias[at]) y += a.bias_value[t.bias[at] - 1];
    // a finite logit stays finite
    if (fabsf(x) <= FLT_MAX) y = fmin(fmax(y, -(double)MOST), (double)MOST);
    return (float)y;
  };

  for (int j = 0; j < rows; ++j) {
    const int64_t row = row0 + j;
    const In* in = static_cast<const In*>(a.logits) + row * a.row_stride + v0;
    Out* out = static_cast<Out*>(a.out) + row * a.out_stride + v0;
    const uint32_t* words = MASK ? a.allowed + row * a.allowed_stride + (v0 >> 5) : nullptr;
    float fill = a.fill;
    if (MASK) {
      // A row that allows nothing at all is -inf throughout, so that no law of it
      // passes for one: looked up only where this chunk allows nothing.
      const int last = (n - 1) >> 5;
      auto any = [&](const uint32_t* w, int end, int bits) {         // words w[0 .. end], `bits` bits of the last
        int hit = 0;
        for (int i = tid; i <= end; i += LC_THREADS) hit |= (w[i] & (i < end || bits == 32 ? ~0u : (1u << bits) - 1u)) != 0u;
        return __syncthreads_or(hit);
      };
      if (!any(words, last, n - 32 * last)) {
        const int end = (a.vocab - 1) >> 5;
        if (!any(words - (v0 >> 5), end, a.vocab - 32 * end)) fill = -INFINITY;
      }
    }
    // 16-byte groups of the row from its first aligned value on; values before and
    // behind them one by one.
    int lead = (int)((16 - ((uintptr_t)in & 15)) & 15) / (int)sizeof(In);
    const bool together = ((uintptr_t)(out + lead) & 15) == 0;
    lead = together ? min(lead, n) : n;
    const int groups = (n - lead) / VEC;
    for (int i = tid; i < groups; i += LC_THREADS) {
      const int at = lead + VEC * i;
      uint32_t keep = (1u << VEC) - 1u;
      if (MASK) keep = bits_from<VEC>(words, at);
      const uint32_t look = bits_from<VEC>(t.touched, at) & keep;
      float x[VEC];
      if (IN == 0) {
        const bf16x8 v = *reinterpret_cast<const bf16x8*>(in + at);
        #pragma unroll
        for (int u = 0; u < VEC; ++u) x[u] = (float)v[u & 7];
      } else {
        const f32x4 v = *reinterpret_cast<const f32x4*>(in + at);
        #pragma unroll
        for (int u = 0; u < VEC; ++u) x[u] = v[u & 3];
      }
      if (look) {
        #pragma unroll
        for (int u = 0; u < VEC; ++u)
          if (look >> u & 1u) x[u] = control(x[u], at + u, j);
      }
      #pragma unroll
      for (int u = 0; u < VEC; ++u) x[u] = keep >> u & 1u ? x[u] : fill;
      if (OUT == 0) {
        bf16x8 v;
        #pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = (bf16)x[u % VEC];
        *reinterpret_cast<bf16x8*>(out + at) = v;
      } else {
        #pragma unroll
        for (int q = 0; q < VEC / 4; ++q)
          *reinterpret_cast<f32x4*>(out + at + 4 * q) = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
      }
    }
    auto single = [&](int at) {
      const bool keep = !MASK || (words[at >> 5] >> (at & 31) & 1u);
      float x = (float)in[at];
      if (t.touched[at >> 5] >> (at & 31) & 1u) x = control(x, at, j);
      out[at] = (Out)(keep ? x : fill);
    };
    for (int at = tid; at < lead; at += LC_THREADS) single(at);
    for (int at = lead + VEC * groups + tid; at < n; at += LC_THREADS) single(at);
  }
}

}  // namespace dspark

using namespace dspark;

namespace {

template <int IN, int OUT>
int launch_controls(const ControlArgs& a, hipStream_t s) {
  constexpr int CH = 4096;
  const dim3 grid((unsigned)((a.vocab + CH - 1) / CH), (unsigned)a.n_req);
  if (a.allowed) hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, true>), grid, dim3(LC_THREADS), 0, s, a);
  else hipLaunchKernelGGL((logit_controls_kernel<IN, OUT, CH, false>), grid, dim3(LC_THREADS), 0, s, a);
  return launch_status("logit_controls_kernel");
}

}  // namespace

extern "C" int dspark_logit_controls(const void* logits, int dtype, int64_t row_stride, int vocab,
                                     const int32_t* cu_rows, int n_req, const int32_t* text, const void* history,
                                     int history_bytes, int64_t history_stride, const int64_t* tokens,
                                     const double* penalties, const int32_t* bias_start, const int32_t* bias_token,
                                     const double* bias_value, const int32_t* allowed, int64_t allowed_stride, float fill,
                                     void* out, int out_dtype, int64_t out_stride, void* stream) {
  clear_error();
  DSPARK_REQUIRE(logits && cu_rows && text && history && penalties && bias_start && out, "null pointer argument");
  DSPARK_REQUIRE(n_req >= 1 && n_req <= 65535, "n_req must be in [1, 65535] (got %d)", n_req);
  DSPARK_REQUIRE(vocab >= 1 && row_stride >= vocab && out_stride >= vocab, "need vocab >= 1 and row strides of at least vocab");
  DSPARK_REQUIRE(dtype == 0 || dtype == 1, "dtype must be 0 (bf16) or 1 (fp32)");
  DSPARK_REQUIRE(out_dtype == 1 || out_dtype == dtype, "out_dtype must be the logits' or 1 (fp32)");
  DSPARK_REQUIRE(history_bytes == 4 || history_bytes == 8, "history must be int32 or int64");
  DSPARK_REQUIRE(history_stride >= 0 && (!allowed || allowed_stride >= (vocab + 31) / 32), "a mask row needs ceil(vocab / 32) words");
  DSPARK_REQUIRE(logits != out || (dtype == out_dtype && row_stride == out_stride), "in place needs one type and row stride");
  ControlArgs a{logits, out, row_stride, out_stride, cu_rows, text, history, history_stride, tokens, penalties, bias_start,
                bias_token, bias_value, reinterpret_cast<const uint32_t*>(allowed), allowed_stride, fill, n_req, vocab,
                history_bytes == 8};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == 1) return launch_controls<1, 1>(a, s);
  return out_dtype == 1 ? launch_controls<0, 1>(a, s) : launch_controls<0, 0>(a, s);
}
