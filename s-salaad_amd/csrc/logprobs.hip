// Log probabilities of given tokens, the entropy and the top alternatives, one
// workgroup a row of logits:
//   d_i = x_i − max x,  S = Σ exp(d_i),  T = Σ exp(d_i)·d_i
//   logprob = d_token − log S,  entropy = log S − T / S
// One pass over the row: each thread keeps a running maximum of its elements
// and S and T relative to it, scaled (without a branch: some lane of a wave meets
// a new maximum in almost every group) once a group of vectors. S is summed in
// 64 bits, so that a row with one likely token keeps the digits of log S near
// zero; a group's terms of T, where the maximum itself adds nothing, are summed
// in fp32 and then in 64 bits.
//
// The alternatives are ordered by a 64-bit key, the logit's bits in an
// order-preserving form over the inverted index: larger logits first, equal ones
// by ascending index, no two keys alike. The top-th largest of the threads' own
// best keys bounds the answer from below, and only threads whose best reaches it
// hold candidates, so that only those read their elements again.
//
// Many rows are bound by memory: 2000 rows of 32000 fp32 logits, 5 alternatives:
// 49 µs a launch, 5.2 TB/s (a copy, which also writes: 4.83). Few rows are bound by
// latency, long ones by the one compute unit that works on each: 16 rows of 32000
// bf16, 8 alternatives: 9.5 µs. Several workgroups a row would need a second launch
// to join them, or a counter kept between calls.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

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

// NaN counts as the largest, below a key of all ones, which stands for none; −0
// equals +0.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.f);
  uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (x != x) o = 0xfffffffeu;
  return ((uint64_t)o << 32) | (0xffffffffu - (uint32_t)i);
}

__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

// The value of lane (l ^ O), for a wave's exchanges without LDS: quads, then
// mirrored halves and rows (l ^ 4 = l ^ 7 ^ 3, l ^ 8 = l ^ 15 ^ 7), then swaps of
// rows and halves.
template <int O>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  constexpr int kQuadRev = 0x1b, kHalfMirror = 0x141, kMirror = 0x140;
  const auto dpp = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true);
  };
  if constexpr (O == 1) return dpp(v, std::integral_constant<int, 0xb1>{});
  else if constexpr (O == 2) return dpp(v, std::integral_constant<int, 0x4e>{});
  else if constexpr (O == 4)
    return dpp(dpp(v, std::integral_constant<int, kHalfMirror>{}),
               std::integral_constant<int, kQuadRev>{});
  else if constexpr (O == 8)
    return dpp(dpp(v, std::integral_constant<int, kMirror>{}),
               std::integral_constant<int, kHalfMirror>{});
  else if constexpr (O == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int O, typename T>
__device__ __forceinline__ T lane_xor(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, lane_xor<O>(__builtin_bit_cast(uint32_t, v)));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(T, ((uint64_t)lane_xor<O>((uint32_t)(u >> 32)) << 32) |
                                     lane_xor<O>((uint32_t)u));
  }
}

// f over the wave's values, in a fixed order
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T v, F f) {
  v = f(v, lane_xor<1>(v));
  v = f(v, lane_xor<2>(v));
  v = f(v, lane_xor<4>(v));
  v = f(v, lane_xor<8>(v));
  v = f(v, lane_xor<16>(v));
  return f(v, lane_xor<32>(v));
}

// One step of a descending bitonic sort over a wave.
template <int SIZE, int O>
__device__ __forceinline__ void sort_step(uint64_t& k, int lane) {
  const uint64_t other = lane_xor<O>(k);
  const bool greater = ((lane & O) == 0) == ((lane & SIZE) == 0);
  k = (k > other) == greater ? k : other;
}
template <int SIZE, int O = SIZE / 2>
__device__ __forceinline__ void sort_wave(uint64_t& k, int lane) {
  if constexpr (SIZE > 2 && O == SIZE / 2) sort_wave<SIZE / 2>(k, lane);
  sort_step<SIZE, O>(k, lane);
  if constexpr (O > 1) sort_wave<SIZE, O / 2>(k, lane);
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
  __device__ __forceinline__ uint4 raw(int v) const {
    return *(const uint4*)(x + peel * Elem<DT>::bytes + (int64_t)v * 16);
  }
  __device__ __forceinline__ void vec(float* f, int v) const { unpack16<DT>(f, raw(v)); }
  __device__ __forceinline__ float at(int i) const { return load_scalar<DT>(x, i); }
};

// A thread's running maximum (and the first element that holds it), S and T. The
// maximum starts at the lowest finite value, below which only −inf lies (whose
// weight is 0 against it).
struct Running {
  float m = -3.402823466e38f;
  int first = -1;
  double S = 0, T = 0;
  // N elements; index(e) is that of the e-th, ascending
  template <int N, typename F>
  __device__ __forceinline__ void add(const float* x, F index) {
    float top = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
    int at = 0;
#pragma unroll
    for (int e = N - 1; e > 0; --e) at = x[e] == top ? e : at;
    at = x[0] == top ? 0 : at;
    if (top > m || (S == 0 && top == m)) first = index(at);
    // finite, so that an S of 0 adds 0
    const float shift = fmaxf(m - fmaxf(m, top), -3.402823466e38f);
    const double f = __builtin_amdgcn_exp2f(shift * 1.44269504f);
    T = f * fma(S, (double)shift, T);
    S *= f;
    m = fmaxf(m, top);
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

// The 64 largest keys of the workgroup's waves (k: each wave's, descending over
// its lanes), descending in lists[0 .. 64). Two lists' largest are the larger of
// one and the other reversed, a bitonic sequence.
template <int NW>
__device__ __forceinline__ void merge_waves(uint64_t k, uint64_t* lists, int wave, int lane) {
  lists[wave * 64 + lane] = k;
#pragma unroll
  for (int n = NW / 2; n > 0; n >>= 1) {
    __syncthreads();
    if (wave < n) {
      const uint64_t other = lists[(wave + n) * 64 + 63 - lane];
      k = k > other ? k : other;
      sort_step<64, 32>(k, lane);
      sort_step<64, 16>(k, lane);
      sort_step<64, 8>(k, lane);
      sort_step<64, 4>(k, lane);
      sort_step<64, 2>(k, lane);
      sort_step<64, 1>(k, lane);
      lists[wave * 64 + lane] = k;
    }
  }
  __syncthreads();
}

template <int DT, int NT>
__global__ __launch_bounds__(NT) void logprobs_kernel(LogprobArgs A) {
  constexpr int VE = Row<DT>::VE, NW = NT / 64;
  const Row<DT> R(A);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t tok = A.tokens[blockIdx.x];
  const bool in = tok >= 0 && tok < A.vocab;
  const float x_tok = R.at(in ? (int)tok : 0);  // early, beside the row
  constexpr int U = 16 / VE * 2;  // vectors of a group: 32 elements, loaded together
  Running own;
  if (tid < R.peel) {
    const float x = R.at(tid);
    own.add<1>(&x, [&](int) { return tid; });
  }
  int v = tid;
  const auto index = [&](int e) { return R.peel + (v + e / VE * NT) * VE + e % VE; };
  // groups of U vectors, the next one's loads before the work on this one; the
  // last has places left out
  uint4 ahead[U];
  const auto load = [&](int first) {
#pragma unroll
    for (int u = 0; u < U; ++u) ahead[u] = R.raw(min(first + u * NT, R.vecs - 1));
  };
  if (v < R.vecs) load(v);
  while (v < R.vecs) {
    float x[U * VE];
#pragma unroll
    for (int u = 0; u < U; ++u) unpack16<DT>(x + u * VE, ahead[u]);
    const int last = v + (U - 1) * NT;
    if (v + U * NT < R.vecs) load(v + U * NT);
    if (last >= R.vecs) {
#pragma unroll
      for (int u = 1; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VE; ++e)
          x[u * VE + e] = v + u * NT < R.vecs ? x[u * VE + e] : -INFINITY;
    }
    own.add<U * VE>(x, index);
    v += U * NT;
  }
  if (tid < R.tail) {
    const int i = A.vocab - R.tail + tid;
    const float x = R.at(i);
    own.add<1>(&x, [&](int) { return i; });
  }
  // the row's maximum, then S and T against it
  __shared__ float wave_m[NW];
  __shared__ double wave_s[NW], wave_t[NW];
  const float w_m = wave_reduce(own.m, [](float a, float b) { return fmaxf(a, b); });
  if (lane == 0) wave_m[wave] = w_m;
  __syncthreads();
  float best = wave_m[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) best = fmaxf(best, wave_m[w]);
  const float shift = fmaxf(own.m - best, -3.402823466e38f);
  const double f = __builtin_amdgcn_exp2f(shift * 1.44269504f);
  const auto sum = [](double a, double b) { return a + b; };
  const double w_s = wave_reduce(f * own.S, sum);
  const double w_t = wave_reduce(f * fma(own.S, (double)shift, own.T), sum);
  if (lane == 0) {
    wave_s[wave] = w_s;
    wave_t[wave] = w_t;
  }
  __syncthreads();
  double S = wave_s[0], T = wave_t[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    S += wave_s[w];
    T += wave_t[w];
  }
  const double log_s = log(S);
  if (tid == 0) {
    A.logprob[blockIdx.x] = in ? (float)((double)(x_tok - best) - log_s) : NAN;
    A.entropy[blockIdx.x] = (float)(log_s - T / S);
  }
  if (A.top == 0) return;
  int64_t* ids = A.ids + (int64_t)blockIdx.x * A.top;
  float* lps = A.top_logprobs + (int64_t)blockIdx.x * A.top;

  __shared__ uint64_t heads[NT];  // the threads' best keys
  __shared__ uint64_t found[kCandidates];
  __shared__ int n_found;
  bool plain = S != S;  // a row with NaN or +inf: the threads' maxima do not order it
  if (!plain) {
    uint64_t k = 0;
    if (own.first >= 0) {
      k = key_of(own.m, own.first);
    } else {  // nothing above −inf: its first element
      const int first = tid < R.peel ? tid
                        : tid < R.vecs ? R.peel + tid * VE
                        : tid < R.tail ? A.vocab - R.tail + tid : -1;
      if (first >= 0) k = key_of(-INFINITY, first);
    }
    if (tid == 0) n_found = 0;
    sort_wave<64>(k, lane);
    merge_waves<NW>(k, heads, wave, lane);
    const uint64_t least = heads[A.top - 1];
    const auto keep = [&](float x, int i) {
      const uint64_t c = key_of(x, i);
      if (c >= least) {
        const int at = atomicAdd(&n_found, 1);
        if (at < kCandidates) found[at] = c;
      }
    };
    // each of the threads that reach it, by a wave
    for (int r = wave; r < A.top; r += NW) {
      const uint64_t head = heads[r];
      if (head == 0) break;
      const int i = index_of(head), vec = (i - R.peel) / VE;
      const int t = i < R.peel ? i : vec < R.vecs ? vec % NT : i - (A.vocab - R.tail);
      if (lane == 0 && t < R.peel) keep(R.at(t), t);
      if (lane == 1 && t < R.tail) keep(R.at(A.vocab - R.tail + t), A.vocab - R.tail + t);
      for (int u = t + lane * NT; u < R.vecs; u += 64 * NT) {
        float x[VE];
        R.vec(x, u);
#pragma unroll
        for (int e = 0; e < VE; ++e) keep(x[e], R.peel + u * VE + e);
      }
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
      const auto larger = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
      k = wave_reduce(k, larger);
      __syncthreads();
      if (lane == 0) heads[wave] = k;
      __syncthreads();
      last = heads[0];
      for (int w = 1; w < NW; ++w) last = larger(last, heads[w]);
      if (tid == 0) {
        ids[r] = index_of(last);
        lps[r] = (float)((double)(R.at(index_of(last)) - best) - log_s);
      }
    }
  }
}

template <int DT, int NT>
void launch_threads(const LogprobArgs& A, int64_t rows, hipStream_t st) {
  hipLaunchKernelGGL((logprobs_kernel<DT, NT>), dim3((unsigned)rows), dim3(NT), 0, st, A);
}

// Threads a row: 512 where rows leave compute units idle and are long (16 rows of
// 32000 bf16, 8 alternatives: 9.6 µs, with 256 10.4), 128 where many are short
// (1966 of 295: 12 µs, with 256 16), else 256 (3 of 19516: 7.8 µs, with 512 8.6;
// 2000 of 32000 fp32: 50 µs, with 512 53).
template <int DT>
void launch_logprobs(const LogprobArgs& A, int64_t rows, hipStream_t st) {
  if (rows <= device_cus() && A.vocab > 24576) launch_threads<DT, 512>(A, rows, st);
  else if (rows > device_cus() && A.vocab <= 1024) launch_threads<DT, 128>(A, rows, st);
  else launch_threads<DT, 256>(A, rows, st);
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
