// Attention over a paged key/value cache: one new token per sequence, or
// chunks of tokens at the ends of their sequences.
//
//   out[t, h] = Σ_j softmax_j(q[t, h]·k_j · scale) · v_j,
//   j <= p and (window == 0 or j > p − window or j < sinks)
//
// The softmax is taken online: a running maximum m, sum l and output o per row,
// o and l scaled by exp(m_old − m_new) where the maximum grows. Scores are kept
// in base 2 (scale · log2 e), all sums in fp32, one rounding at the store.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "paged.h"

namespace ssl {
namespace {

// The token's sequence, by bisection of cu (the last s with cu[s] <= t; seqs
// for tokens past the last).
__device__ __forceinline__ int seq_of(const int32_t* cu, int seqs, int64_t t) {
  int lo = 0, hi = seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// One wave a (token, head): lane i scores position i of a run of 64, the
// outputs' features are spread over the lanes.
template <int DT, int HD>
__global__ __launch_bounds__(64) void attn_row_kernel(PagedCache C, AttnArgs A) {
  constexpr int F = HD / 64;
  __shared__ float qs[HD];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, lane = threadIdx.x;
  const int kh = h / (A.heads / C.kv_heads);
  int s = (int)t;
  int64_t len = 0, p = -1;
  if (A.cu) s = seq_of(A.cu, C.seqs, t);
  if (s < C.seqs) {
    len = min(max((int64_t)A.lengths[s], (int64_t)0), (int64_t)C.cols * C.page);
    p = A.cu ? len - A.cu[s + 1] + t : len - 1;
  }
  for (int f = 0; f < F; ++f)
    qs[lane * F + f] =
        load_scalar<DT>(A.q, t * A.q_token + h * A.q_head + lane * F + f) * A.scale_log2;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[F];
  for (int f = 0; f < F; ++f) o[f] = 0.f;
  const int64_t first = A.window ? max(p + 1 - A.window, (int64_t)0) : 0;
  for (int64_t j0 = 0; j0 <= p; j0 += 64) {
    if (j0 + 64 <= first && j0 >= A.sinks) continue;
    const int64_t j = j0 + lane;
    int64_t off = -1;
    if (j <= p && (j >= first || j < A.sinks)) {
      const int32_t page = C.table[s * C.table_stride + (j >> C.log2_page)];
      if (C.has(page))
        off = page * C.page_stride + kh * C.head_stride + (j & (C.page - 1)) * C.slot_stride;
    }
    float x = -INFINITY;
    if (off >= 0) {
      x = 0.f;
      for (int d = 0; d < HD; ++d) x += qs[d] * load_scalar<DT>(C.k, off + d);
    }
    float mx = x;
    for (int k = 1; k < 64; k <<= 1) mx = fmaxf(mx, __shfl_xor(mx, k));
    const float mn = fmaxf(m, mx);
    if (mn == -INFINITY) continue;
    const float a = exp2f(m - mn), e = off >= 0 ? exp2f(x - mn) : 0.f;
    float sum = e;
    for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
    l = l * a + sum;
    m = mn;
    for (int f = 0; f < F; ++f) o[f] *= a;
    for (int k = 0; k < 64; ++k) {
      const float e_k = __shfl(e, k);
      const int64_t off_k = __shfl((long long)off, k);
      if (off_k < 0) continue;
      for (int f = 0; f < F; ++f) o[f] += e_k * load_scalar<DT>(C.v, off_k + lane * F + f);
    }
  }
  for (int f = 0; f < F; ++f) {
    const float r = l > 0.f ? o[f] / l : (l == 0.f ? 0.f : l);
    const int64_t i = (t * A.heads + h) * HD + lane * F + f;
    if constexpr (DT == DT_F32) ((float*)A.out)[i] = r;
    else ((uint16_t*)A.out)[i] = (uint16_t)to_bits<DT>(r);
  }
}

template <int DT>
void launch_rows(const PagedCache& C, const AttnArgs& A, hipStream_t st) {
  const dim3 grid((unsigned)A.tokens, (unsigned)A.heads);
  if (C.head_dim == 64) hipLaunchKernelGGL((attn_row_kernel<DT, 64>), grid, dim3(64), 0, st, C, A);
  else if (C.head_dim == 128) hipLaunchKernelGGL((attn_row_kernel<DT, 128>), grid, dim3(64), 0, st, C, A);
  else hipLaunchKernelGGL((attn_row_kernel<DT, 256>), grid, dim3(64), 0, st, C, A);
}

}  // namespace
}  // namespace ssl

using namespace ssl;

namespace ssl {
namespace {

// Checks the arguments and fills the kernels' form of them; `need` receives the
// workspace the call takes.
int attention_args(const ssl_paged_attention_args* a, PagedCache* C, AttnArgs* A, int64_t* need) {
  const char* what = "paged_attention";
  *need = 0;
  if (!a) return fail(SSL_ERR_INVALID, "%s: no arguments", what);
  if (int rc = paged_cache(what, a->cache, sizeof(*a), true, C)) return rc;
  if (a->tokens < 0 || a->tokens > 0x7fffffff || a->heads <= 0 || a->heads > 65535 ||
      a->heads % C->kv_heads)
    return fail(SSL_ERR_INVALID, "%s: %lld tokens, %lld heads over %d key/value heads", what,
                (long long)a->tokens, (long long)a->heads, C->kv_heads);
  if (a->window < 0 || a->sinks < 0 || a->max_tokens < 0 || a->max_length < 0)
    return fail(SSL_ERR_INVALID, "%s: window %lld, sinks %lld, at most %lld tokens and %lld positions",
                what, (long long)a->window, (long long)a->sinks, (long long)a->max_tokens,
                (long long)a->max_length);
  if (!a->cu && a->tokens != C->seqs)
    return fail(SSL_ERR_INVALID, "%s: %lld tokens for %d sequences", what, (long long)a->tokens,
                C->seqs);
  if (a->tokens == 0) return SSL_OK;
  if (!a->cu && a->tokens > 65535)
    return fail(SSL_ERR_UNSUPPORTED, "%s: %lld sequences in one call (at most 65535)", what,
                (long long)a->tokens);
  if (!a->q || !a->out || (!a->lengths && C->seqs))
    return fail(SSL_ERR_INVALID, "%s: null pointer", what);
  const int64_t eb = elem_bytes((int)a->cache.dtype);
  if (!aligned(a->q, 16) || !aligned(a->out, 16) || (a->q_token * eb) % 16 || (a->q_head * eb) % 16)
    return fail(SSL_ERR_INVALID, "%s: q's rows and out must be 16-byte aligned", what);
  // lane offsets within a page's head are 32-bit
  if (C->page * C->slot_stride * eb > 0x7fffffff)
    return fail(SSL_ERR_UNSUPPORTED, "%s: a page's head spans 2 GiB or more", what);
  *A = AttnArgs{};
  A->q = (const char*)a->q;
  A->q_token = a->q_token;
  A->q_head = a->q_head;
  A->out = (char*)a->out;
  A->lengths = a->lengths;
  A->cu = a->cu;
  A->tokens = a->tokens;
  A->heads = (int)a->heads;
  // positions are below 2^31, so larger values mean the same as these
  A->window = (int)std::min<int64_t>(a->window, 0x7fffffff);
  A->sinks = (int)std::min<int64_t>(a->sinks, 0x7fffffff);
  A->scale_log2 = (float)(a->scale * 1.4426950408889634);
  const int64_t reach = std::min<int64_t>(a->max_length, (int64_t)C->cols * C->page);
  if (!a->cu && C->cols) *need = paged_decode_plan(*C, A, (int)a->cache.dtype, reach);
  return SSL_OK;
}

}  // namespace
}  // namespace ssl

extern "C" int64_t ssl_paged_attention_workspace_size(const ssl_paged_attention_args* a) {
  PagedCache C;
  AttnArgs A;
  int64_t need;
  return attention_args(a, &C, &A, &need) == SSL_OK ? need : 0;
}

extern "C" int ssl_paged_attention(const ssl_paged_attention_args* a, void* stream) {
  clear_error();
  PagedCache C;
  AttnArgs A;
  int64_t need;
  if (int rc = attention_args(a, &C, &A, &need)) return rc;
  if (a->tokens == 0) return SSL_OK;
  if (need) {
    if (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16))
      return fail(SSL_ERR_WORKSPACE, "paged_attention: workspace of %lld bytes needed",
                  (long long)need);
    A.part_o = (float*)a->workspace;
    A.part_ml = A.part_o + need / 4 / (C.head_dim + 2) * C.head_dim;
  }
  hipStream_t st = (hipStream_t)stream;
  if (!a->cu && C.cols) return paged_decode_launch(C, A, (int)a->cache.dtype, st);
  if (a->cache.dtype == SSL_F32) launch_rows<DT_F32>(C, A, st);
  else if (a->cache.dtype == SSL_BF16) launch_rows<DT_BF16>(C, A, st);
  else launch_rows<DT_F16>(C, A, st);
  return check_hip(hipGetLastError(), "paged_attention launch");
}
