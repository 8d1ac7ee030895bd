// What the kernels over a paged key/value cache share: the cache as they see
// it and the host's checks of the caller's description.
#pragma once

#include <atomic>

#include "abi_internal.h"
#include "slr_common.h"

namespace ssl {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Strides in elements. A page number read from the table is used only after
// `has` accepted it.
struct PagedCache {
  char *k, *v;
  int64_t layer_stride, page_stride, head_stride, slot_stride;
  int64_t pages;
  const int32_t* table;
  int64_t table_stride;
  int layers, kv_heads, page, log2_page, head_dim;
  int seqs, cols;

  __device__ __forceinline__ bool has(int32_t page_no) const {
    return (uint32_t)page_no < (uint32_t)pages;
  }
};

// Checks `c` (the pools only where `pools`) and fills `out`.
int paged_cache(const char* what, const ssl_paged_cache& c, int64_t struct_bytes, bool pools,
                PagedCache* out);

struct AttnArgs {
  const char* q;
  int64_t q_token, q_head;
  char* out;  // [tokens, heads, head_dim]
  const int32_t *lengths, *cu;
  int64_t tokens;
  int heads, window, sinks;
  // |scale| · log2 e (scores are kept in base 2; 1 for a scale whose float is 0), and what
  // its sign does to q: kept bits, flipped sign bits
  float scale_log2;
  uint32_t keep, flip;
  // split contexts: the most parts of a row and its tiles per part at least,
  // and the parts' outputs, maxima and sums
  int n_split, per;
  int waves;  // of a workgroup of the kernel for few rows
  float us;   // the plan's estimate of the call
  float *part_o, *part_ml;
};

// A sequence's rows of one key/value head: its tokens' query heads, packed token
// by token (row r: token r / G, head r % G of the group), and their positions.
struct Chunk {
  int64_t t0;    // its first token
  int rows, p0;  // p0: the first token's position
  __device__ __forceinline__ Chunk(const PagedCache& C, const AttnArgs& A, int s, int G) {
    int64_t a = s, b = s + 1;
    if (A.cu) {
      a = s == 0 ? 0 : A.cu[s];
      a = min(max(a, (int64_t)0), A.tokens);
      b = min(max((int64_t)A.cu[s + 1], a), A.tokens);
    }
    t0 = a;
    rows = (int)(b - a) * G;
    p0 = min(max(A.lengths[s], 0), C.cols << C.log2_page) - (int)(b - a);
  }
  // tokens a … b − 1 of a sequence of `length` positions
  __device__ __forceinline__ Chunk(const PagedCache& C, int a, int b, int length, int G)
      : t0(a), rows((b - a) * G), p0(min(max(length, 0), C.cols << C.log2_page) - (b - a)) {}
  // one token a sequence
  __device__ __forceinline__ Chunk(const PagedCache& C, const AttnArgs& A, int s)
      : t0(s), rows(A.heads / C.kv_heads),
        p0(min(max(A.lengths[s], 0), C.cols << C.log2_page) - 1) {}
};

// Zeros for the heads of key/value head kh of tokens past the last chunk.
__device__ __forceinline__ void zero_tail(const PagedCache& C, const AttnArgs& A, int kh, int row16,
                                          int tid, int threads) {
  const int G = A.heads / C.kv_heads;
  const int64_t end = min(max((int64_t)A.cu[C.seqs], (int64_t)0), A.tokens);
  const int64_t n = (A.tokens - end) * G * row16;
  for (int64_t i = tid; i < n; i += threads) {
    const int64_t r = i / row16;
    *(uint4*)(A.out + (((end + r / G) * A.heads + kh * G + r % G) * row16 + i % row16) * 16) =
        uint4{0, 0, 0, 0};
  }
}

// The positions a run of tokens at p_min … p_max of one sequence sees, as tiles
// of T positions: the first `sink_tiles` of the context, then those from `base`.
struct TileRange {
  int sink_tiles, base, count;
  __device__ __forceinline__ int tile(int i) const {
    return i < sink_tiles ? i : i - sink_tiles + base;
  }
};
template <int T>
__device__ __forceinline__ TileRange tile_range(int p_min, int p_max, int window, int sinks) {
  TileRange r{0, 0, 0};
  if (p_max < 0) return r;
  const int first = window && p_min + 1 > window ? p_min + 1 - window : 0;
  r.base = first / T;
  if (first > 0) r.sink_tiles = min((min(sinks, first) + T - 1) / T, r.base);
  r.count = r.sink_tiles + p_max / T + 1 - r.base;
  return r;
}

// The tiles a part of a row takes: A.per, or what spreads `count` over the
// most parts. The kernels and the join compute the same.
__device__ __forceinline__ int part_tiles(const AttnArgs& A, int count) {
  return max(A.per, (count + A.n_split - 1) / A.n_split);
}

// Bits of two adjacent 16-bit elements, p rounded to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == DT_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// The 16-bit element in the low half of x.
template <int DT>
__device__ __forceinline__ float low16(uint32_t x) {
  return DT == DT_BF16 ? bf16_to_f32(x & 0xffffu) : f16_to_f32(x & 0xffffu);
}

// A product rounded before it is used (and not fused into what uses it).
__device__ __forceinline__ float rounded(float x) {
  asm("" : "+v"(x));
  return x;
}
// From here on the prompt kernel's weights take rounded scores. (Below, a fused
// product minus the rounded maximum is off by at most 2^-4 in the exponent, for all
// of a row alike; above, a half step of the maximum would overflow the weights.)
constexpr float kFarScore = 1048576.f;

// Lets `kernel` take `bytes` of dynamic shared memory on the current device; `raised`
// holds a bit a device on which it may, and starts at 0.
int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>* raised);

// Few rows of a key/value head (paged_decode.hip), or many (paged_prompt.hip).
// The plans fill the split and return the bytes of the parts.
int64_t paged_decode_plan(const PagedCache& C, AttnArgs* A, int dtype, int64_t max_tokens,
                          int64_t max_length);
int paged_decode_launch(const PagedCache& C, const AttnArgs& A, int dtype, int64_t max_tokens,
                        hipStream_t st);
int64_t paged_prompt_plan(const PagedCache& C, AttnArgs* A, int dtype, int64_t max_tokens,
                          int64_t max_length);
int paged_prompt_launch(const PagedCache& C, const AttnArgs& A, int dtype, hipStream_t st);

}  // namespace ssl
