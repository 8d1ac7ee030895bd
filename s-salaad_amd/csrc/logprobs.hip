// Log probabilities of given tokens, the entropy and the top alternatives, one
// workgroup a row of logits:
//   d_i = x_i − max x,  S = Σ exp(d_i),  T = Σ exp(d_i)·d_i   (sums in 64 bits)
//   logprob = d_token − log S,  entropy = log S − T / S
// The sums are 64-bit so that a row with one likely token keeps the digits of
// log S near zero. The alternatives are ordered by a 64-bit key, the logit's
// bits in an order-preserving form over the inverted index: larger logits
// first, equal ones by ascending index, no two keys alike.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "abi_internal.h"
#include "slr_common.h"

namespace ssl {
namespace {

constexpr int kTopMax = 64;
constexpr int kRowThreads = 256;

struct LogprobArgs {
  const char* x;
  int64_t ld;
  int vocab, top;
  const int64_t* tokens;
  float *logprob, *entropy;
  int64_t* ids;
  float* top_logprobs;
};

// NaN counts as the largest; −0 equals +0.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.f);
  uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (x != x) o = 0xffffffffu;
  return ((uint64_t)o << 32) | (0xffffffffu - (uint32_t)i);
}

template <typename T, typename F>
__device__ __forceinline__ T reduce(T v, F f) {
  __shared__ T part[kRowThreads / 64];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = f(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < kRowThreads / 64; ++w) v = f(v, part[w]);
  return v;
}

template <int DT>
__global__ __launch_bounds__(kRowThreads) void logprobs_kernel(LogprobArgs A) {
  const int64_t row = blockIdx.x, base = row * A.ld;
  const int tid = threadIdx.x;
  float best = -INFINITY;
  for (int i = tid; i < A.vocab; i += kRowThreads) {
    const float x = load_scalar<DT>(A.x, base + i);
    best = x != x || best != best ? NAN : fmaxf(best, x);
  }
  best = reduce(best, [](float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); });
  double s = 0, t = 0;
  for (int i = tid; i < A.vocab; i += kRowThreads) {
    const float d = load_scalar<DT>(A.x, base + i) - best;
    const float e = expf(d);
    s += e;
    if (!(e == 0.f)) t += (double)e * d;
  }
  s = reduce(s, [](double a, double b) { return a + b; });
  t = reduce(t, [](double a, double b) { return a + b; });
  const double log_s = log(s);
  if (tid == 0) {
    const int64_t tok = A.tokens[row];
    const bool in = tok >= 0 && tok < A.vocab;
    A.logprob[row] = in ? (float)((double)(load_scalar<DT>(A.x, base + tok) - best) - log_s) : NAN;
    A.entropy[row] = (float)(log_s - t / s);
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < A.top; ++r) {
    uint64_t k = 0;
    for (int i = tid; i < A.vocab; i += kRowThreads) {
      const uint64_t c = key_of(load_scalar<DT>(A.x, base + i), i);
      if (c < last && c > k) k = c;
    }
    last = reduce(k, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    if (tid == 0) {
      const int64_t i = 0xffffffffu - (uint32_t)last;
      A.ids[row * A.top + r] = i;
      A.top_logprobs[row * A.top + r] =
          (float)((double)(load_scalar<DT>(A.x, base + i) - best) - log_s);
    }
  }
}

}  // namespace
}  // namespace ssl

using namespace ssl;

extern "C" int ssl_token_logprobs(const ssl_token_logprobs_args* a, void* stream) {
  clear_error();
  const char* what = "token_logprobs";
  if (!a || a->bytes != (int64_t)sizeof(*a))
    return fail(SSL_ERR_INVALID, "%s: no arguments, or of another size", what);
  if (a->dtype != SSL_F32 && a->dtype != SSL_BF16 && a->dtype != SSL_F16)
    return fail(SSL_ERR_UNSUPPORTED, "%s: unknown dtype code %lld", what, (long long)a->dtype);
  if (a->rows < 0 || a->rows > 0x7fffffff || a->vocab <= 0 || a->vocab > 0x7fffffff ||
      a->ld < a->vocab)
    return fail(SSL_ERR_INVALID, "%s: %lld rows of %lld logits, %lld apart", what,
                (long long)a->rows, (long long)a->vocab, (long long)a->ld);
  if (a->top < 0 || a->top > a->vocab || a->top > kTopMax)
    return fail(SSL_ERR_INVALID, "%s: top %lld of %lld (at most %d)", what, (long long)a->top,
                (long long)a->vocab, kTopMax);
  if (a->rows == 0) return SSL_OK;
  if (!a->logits || !a->tokens || !a->logprob || !a->entropy ||
      (a->top && (!a->top_ids || !a->top_logprobs)))
    return fail(SSL_ERR_INVALID, "%s: null pointer", what);
  LogprobArgs A{(const char*)a->logits, a->ld, (int)a->vocab, (int)a->top, a->tokens, a->logprob,
                a->entropy, a->top_ids, a->top_logprobs};
  const dim3 grid((unsigned)a->rows);
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == SSL_F32) hipLaunchKernelGGL(logprobs_kernel<DT_F32>, grid, dim3(kRowThreads), 0, st, A);
  else if (a->dtype == SSL_BF16) hipLaunchKernelGGL(logprobs_kernel<DT_BF16>, grid, dim3(kRowThreads), 0, st, A);
  else hipLaunchKernelGGL(logprobs_kernel<DT_F16>, grid, dim3(kRowThreads), 0, st, A);
  return check_hip(hipGetLastError(), "token_logprobs launch");
}
