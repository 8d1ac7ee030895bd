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

using namespace ssl;

namespace ssl {

int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>* raised) {
  int dev = 0;
  if (int rc = check_hip(hipGetDevice(&dev), "device query")) return rc;
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (raised->load(std::memory_order_relaxed) & bit) return SSL_OK;
  if (int rc = check_hip(
          hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
          "shared memory size"))
    return rc;
  raised->fetch_or(bit, std::memory_order_relaxed);
  return SSL_OK;
}

namespace {

// Rows of one key/value head the kernel for few of them is considered for, which
// reads a context once for 16. (500 tokens, 8 fp32 heads of 128: 20 µs, the other
// 34; 8 chunks of 40 over 8000 positions, 16 heads of 64: 55 µs, the other 48. In
// 16 bits more rows are never its case: 300 tokens of a group of 4 over 2000
// positions 26 µs, the other 20.)
constexpr int few_rows(int dtype) { return dtype == SSL_F32 ? 4096 : 512; }

// Checks the arguments and fills the kernels' form of them; `need` receives the
// workspace the call takes, `few` which kernel.
int attention_args(const ssl_paged_attention_args* a, PagedCache* C, AttnArgs* A, int64_t* need,
                   bool* few) {
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
  if (a->tokens * a->heads > 0x7fffffffLL)
    return fail(SSL_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads in one call", what,
                (long long)a->tokens, (long long)a->heads);
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
  if (!(fabs(a->scale) < 1e30))
    return fail(SSL_ERR_INVALID, "%s: scale %g", what, a->scale);
  // (a scale whose float is 0 is one of 0, not a product of it with a masked −inf)
  const float scale = (float)(fabs(a->scale) * 1.4426950408889634);
  A->scale_log2 = scale == 0 ? 1.f : scale;
  A->keep = scale == 0 ? 0u : ~0u;
  A->flip = a->scale < 0 ? ~0u : 0u;
  const int64_t reach = std::min<int64_t>(a->max_length, (int64_t)C->cols * C->page);
  if (C->cols == 0) return fail(SSL_ERR_INVALID, "%s: a table without columns", what);
  const int dtype = (int)a->cache.dtype;
  const int64_t most = a->cu ? std::min<int64_t>(a->max_tokens, a->tokens) : 1;
  const int64_t rows = most * (A->heads / C->kv_heads);
  *few = !a->cu;
  if (a->cu) {
    *need = paged_prompt_plan(*C, A, dtype, most, reach);
    if (rows <= few_rows(dtype) && C->seqs < 65535 && C->kv_heads * ((rows + 15) / 16) <= 65535) {
      AttnArgs other = *A;
      const int64_t bytes = paged_decode_plan(*C, &other, dtype, most, reach);
      if (other.us <= A->us) {
        *few = true;
        *A = other;
        *need = bytes;
      }
    }
  } else {
    *need = paged_decode_plan(*C, A, dtype, most, reach);
  }
  return SSL_OK;
}

}  // namespace
}  // namespace ssl

extern "C" int64_t ssl_paged_attention_workspace_size(const ssl_paged_attention_args* a) {
  PagedCache C;
  AttnArgs A;
  int64_t need;
  bool few;
  return attention_args(a, &C, &A, &need, &few) == SSL_OK ? need : 0;
}

extern "C" int ssl_paged_attention(const ssl_paged_attention_args* a, void* stream) {
  clear_error();
  PagedCache C;
  AttnArgs A;
  int64_t need;
  bool few;
  if (int rc = attention_args(a, &C, &A, &need, &few)) return rc;
  if (a->tokens == 0) return SSL_OK;
  if (need) {
    if (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16))
      return fail(SSL_ERR_WORKSPACE, "paged_attention: workspace of %lld bytes needed",
                  (long long)need);
    A.part_o = (float*)a->workspace;
    A.part_ml = A.part_o + need / 4 / (C.head_dim + 2) * C.head_dim;
  }
  hipStream_t st = (hipStream_t)stream;
  const int64_t most = a->cu ? std::min<int64_t>(a->max_tokens, a->tokens) : 1;
  return few ? paged_decode_launch(C, A, (int)a->cache.dtype, most, st)
             : paged_prompt_launch(C, A, (int)a->cache.dtype, st);
}
