// Log probabilities of given tokens, the entropy and the top alternatives, one
// workgroup a row of logits:
//   d_i = x_i − max x,  S = Σ exp(d_i),  T = Σ exp(d_i)·d_i
//   logprob = d_token − log S,  entropy = log S − T / S
// One pass over the row: each thread keeps a running maximum of its elements
// and S and T relative to it. S is summed in 64 bits, so that a row with one
// likely token keeps the digits of log S near zero; a vector's terms of T, where
// the maximum itself adds nothing, are summed in fp32 and then in 64 bits.
//
// The alternatives are ordered by a 64-bit key, the logit's bits in an
// order-preserving form over the inverted index: larger logits first, equal ones
// by ascending index, no two keys alike. The top-th largest of the threads' own
// best keys bounds the answer from below, and only threads whose best reaches it
// hold candidates, so that only those read their elements again.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "abi_internal.h"
#include "slr_common.h"

namespace ssl {
namespace {

constexpr int kTopMax = 64;

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

__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

// f over the workgroup's values, in a fixed order
template <int NT, typename T, typename F>
__device__ __forceinline__ T reduce(T v, F f) {
  __shared__ T part[NT / 64];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = f(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = f(v, part[w]);
  return v;
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return ((uint64_t)__shfl_xor((uint32_t)(v >> 32), o) << 32) | __shfl_xor((uint32_t)v, o);
}

constexpr int kCandidates = 2048;

template <int DT>
struct Row {
  static constexpr int VE = 16 / Elem<DT>::bytes;
  const char* x;      // the row
  int peel, vecs, tail;  // elements before the first 16-byte boundary, vectors, elements after
  __device__ __forceinline__ Row(const LogprobArgs& A) {
    x = A.x + (int64_t)blockIdx.x * A.ld * Elem<DT>::bytes;
    peel = min((int)((16 - ((uintptr_t)x & 15)) & 15) / Elem<DT>::bytes, A.vocab);
    vecs = (A.vocab - peel) / VE;
    tail = A.vocab - peel - vecs * VE;
  }
  __device__ __forceinline__ void vec(float* f, int v) const {
    const uint4 r = *(const uint4*)(x + peel * Elem<DT>::bytes + (int64_t)v * 16);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == DT_F32) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (DT == DT_BF16) {
        f[2 * i] = bf16_to_f32(w[i] & 0xffffu);
        f[2 * i + 1] = bf16_to_f32(w[i] >> 16);
      } else {
        f[2 * i] = f16_to_f32(w[i] & 0xffffu);
        f[2 * i + 1] = f16_to_f32(w[i] >> 16);
      }
    }
  }
  __device__ __forceinline__ float at(int i) const { return load_scalar<DT>(x, i); }
};

// A thread's running maximum (and its first index), S and T.
struct Running {
  float m = -INFINITY;
  int first = -1;
  double S = 0, T = 0;
  template <int N>
  __device__ __forceinline__ void add(const float* x, int i0) {
    float top = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
    if (!(top <= m)) {  // greater, or NaN throughout
      const float shift = m - top;  // −inf at the first
      if (S != 0) {
        const double f = expf(shift);
        T = f * (T + S * shift);
        S *= f;
      }
      m = top;
#pragma unroll
      for (int e = N - 1; e >= 0; --e)
        if (x[e] == top) first = i0 + e;
    }
    if (m == -INFINITY) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (x[e] != x[e]) S = NAN;
      return;
    }
    float t = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[e] - m;
      const float p = __builtin_amdgcn_exp2f(d * 1.44269504f);
      S += p;
      t = fmaf(p, fmaxf(d, -1e30f), t);  // −inf: 0 · −1e30
    }
    T += t;
  }
};

template <int DT, int NT>
__global__ __launch_bounds__(NT) void logprobs_kernel(LogprobArgs A) {
  constexpr int VE = Row<DT>::VE, NW = NT / 64;
  const Row<DT> R(A);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Running own;
  // a thread of nothing above −inf has its first element for its best
  own.first = tid < R.peel ? tid
              : tid < R.vecs ? R.peel + tid * VE
              : tid < R.tail ? A.vocab - R.tail + tid : -1;
  if (tid < R.peel) {
    const float x = R.at(tid);
    own.add<1>(&x, tid);
  }
  constexpr int U = 4;  // vectors in flight
  int v = tid;
  for (; v + (U - 1) * NT < R.vecs; v += U * NT) {
    float x[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) R.vec(x[u], v + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u) own.add<VE>(x[u], R.peel + (v + u * NT) * VE);
  }
  for (; v < R.vecs; v += NT) {
    float x[VE];
    R.vec(x, v);
    own.add<VE>(x, R.peel + v * VE);
  }
  if (tid < R.tail) {
    const float x = R.at(A.vocab - R.tail + tid);
    own.add<1>(&x, A.vocab - R.tail + tid);
  }
  const float best = reduce<NT>(own.m, [](float a, float b) { return fmaxf(a, b); });
  double S = 0, T = 0;
  if (own.S != 0) {
    const float shift = own.m - best;
    const double f = expf(shift);
    S = f * own.S;
    T = f * (own.T + own.S * shift);
  }
  const auto sum = [](double a, double b) { return a + b; };
  S = reduce<NT>(S, sum);
  T = reduce<NT>(T, sum);
  const double log_s = log(S);
  if (tid == 0) {
    const int64_t tok = A.tokens[blockIdx.x];
    const bool in = tok >= 0 && tok < A.vocab;
    A.logprob[blockIdx.x] = in ? (float)((double)(R.at((int)tok) - best) - log_s) : NAN;
    A.entropy[blockIdx.x] = (float)(log_s - T / S);
  }
  if (A.top == 0) return;
  int64_t* ids = A.ids + (int64_t)blockIdx.x * A.top;
  float* lps = A.top_logprobs + (int64_t)blockIdx.x * A.top;

  __shared__ uint64_t heads[NT];         // each wave's best keys, descending
  __shared__ uint64_t found[kCandidates];
  __shared__ uint64_t bound;
  __shared__ int n_found;
  bool plain = S != S;  // a row with NaN or +inf: the threads' maxima do not order it
  if (!plain) {
    const uint64_t mine = own.first < 0 ? 0 : key_of(own.m, own.first);
    uint64_t k = mine;  // sorted over the wave, descending
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
      for (int o = size >> 1; o > 0; o >>= 1) {
        const uint64_t other = shfl_xor64(k, o);
        const bool greater = ((lane & o) == 0) == ((lane & size) == 0);
        k = greater ? (k > other ? k : other) : (k < other ? k : other);
      }
    heads[tid] = k;
    if (tid == 0) {
      n_found = 0;
      bound = 0;
    }
    __syncthreads();
    if (lane < A.top && k) {  // its rank among all waves' keys
      int rank = lane;
      for (int w = 0; w < NW; ++w) {
        if (w == wave) continue;
        int lo = 0, hi = 64;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (heads[w * 64 + mid] > k) lo = mid + 1;
          else hi = mid;
        }
        rank += lo;
      }
      if (rank == A.top - 1) bound = k;
    }
    __syncthreads();
    const uint64_t least = bound;
    if (mine && mine >= least) {
      auto keep = [&](float x, int i) {
        const uint64_t c = key_of(x, i);
        if (c >= least) {
          const int at = atomicAdd(&n_found, 1);
          if (at < kCandidates) found[at] = c;
        }
      };
      if (tid < R.peel) keep(R.at(tid), tid);
#pragma unroll 4
      for (int u = tid; u < R.vecs; u += NT) {
        float x[VE];
        R.vec(x, u);
#pragma unroll
        for (int e = 0; e < VE; ++e) keep(x[e], R.peel + u * VE + e);
      }
      if (tid < R.tail) keep(R.at(A.vocab - R.tail + tid), A.vocab - R.tail + tid);
    }
    __syncthreads();
    const int n = n_found;
    plain = n > kCandidates;
    if (!plain) {
      for (int i = tid; i < n; i += NT) {
        const uint64_t c = found[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += found[j] > c;
        if (rank < A.top) {
          ids[rank] = index_of(c);
          lps[rank] = (float)((double)(logit_of(c) - best) - log_s);
        }
      }
    }
  }
  if (plain) {  // one pass over the row per alternative
    uint64_t last = ~0ull;
    for (int r = 0; r < A.top; ++r) {
      uint64_t k = 0;
      for (int i = tid; i < A.vocab; i += NT) {
        const uint64_t c = key_of(R.at(i), i);
        if (c < last && c > k) k = c;
      }
      last = reduce<NT>(k, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
      if (tid == 0) {
        ids[r] = index_of(last);
        lps[r] = (float)((double)(R.at(index_of(last)) - best) - log_s);
      }
    }
  }
}

template <int DT>
void launch_logprobs(const LogprobArgs& A, int64_t rows, hipStream_t st) {
  // up to one row a compute unit: every wave it holds works on that row
  if (rows <= device_cus())
    hipLaunchKernelGGL((logprobs_kernel<DT, 1024>), dim3((unsigned)rows), dim3(1024), 0, st, A);
  else
    hipLaunchKernelGGL((logprobs_kernel<DT, 256>), dim3((unsigned)rows), dim3(256), 0, st, A);
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
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == SSL_F32) launch_logprobs<DT_F32>(A, a->rows, st);
  else if (a->dtype == SSL_BF16) launch_logprobs<DT_BF16>(A, a->rows, st);
  else launch_logprobs<DT_F16>(A, a->rows, st);
  return check_hip(hipGetLastError(), "token_logprobs launch");
}
