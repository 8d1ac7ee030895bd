// A paged key/value cache: new tokens written into pages, and pages freed,
// forked and compacted. The attention over them is in paged_attention.hip.
//
//   append      rotary embedding of q and k, k and v into their pages
//   free        sequences' rows cleared, their pages' references taken back
//   fork        sequences that go on as copies of others: whole pages shared,
//               a partly filled last page copied
//   compact     the pages in use moved to the lowest page numbers
//
// The page operations are two launches each (freeing in a small state is one):
// the first settles which pages are taken (one workgroup ranks them; others copy
// the small state arrays), the second moves the data over the whole device.
// Reference counts change by integer atomics, whose order does not change the
// result.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "paged.h"

namespace ssl {

int paged_cache(const char* what, const ssl_paged_cache& c, int64_t struct_bytes, bool pools,
                PagedCache* out) {
  if (c.bytes != struct_bytes)
    return fail(SSL_ERR_INVALID, "%s: an argument struct of %lld bytes, not %lld", what,
                (long long)c.bytes, (long long)struct_bytes);
  if (c.seqs < 0 || c.cols < 0 || c.seqs > 0x7fffffff || c.cols > 0x7fffffff || c.pages <= 0 ||
      c.pages > 0x7fffffff || c.table_stride < c.cols || (c.seqs * c.cols > 0 && !c.table))
    return fail(SSL_ERR_INVALID, "%s: a table of %lld x %lld (stride %lld) over %lld pages", what,
                (long long)c.seqs, (long long)c.cols, (long long)c.table_stride,
                (long long)c.pages);
  *out = PagedCache{(char*)c.k,    (char*)c.v,     c.layer_stride, c.page_stride,
                    c.head_stride, c.slot_stride,  c.pages,        c.table,
                    c.table_stride, (int)c.layers, (int)c.kv_heads, (int)c.page,
                    0,             (int)c.head_dim, (int)c.seqs,    (int)c.cols};
  if (c.page < 16 || c.page > 1024 || (c.page & (c.page - 1)))
    return fail(SSL_ERR_UNSUPPORTED, "%s: page of %lld (a power of two from 16 to 1024)", what,
                (long long)c.page);
  while ((1 << out->log2_page) < out->page) ++out->log2_page;
  // positions are 32-bit
  if (c.cols * c.page > 0x7fffffff)
    return fail(SSL_ERR_INVALID, "%s: %lld columns of %lld positions (below 2^31)", what,
                (long long)c.cols, (long long)c.page);
  if (!pools) return SSL_OK;
  if (c.dtype != SSL_F32 && c.dtype != SSL_BF16 && c.dtype != SSL_F16)
    return fail(SSL_ERR_UNSUPPORTED, "%s: unknown dtype code %lld", what, (long long)c.dtype);
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail(SSL_ERR_UNSUPPORTED, "%s: head_dim %lld (64, 128 or 256)", what,
                (long long)c.head_dim);
  if (c.layers <= 0 || c.layers > 65535 || c.kv_heads <= 0 || c.kv_heads > 65535 || !c.k || !c.v)
    return fail(SSL_ERR_INVALID, "%s: %lld layers of %lld key/value heads, or no pools", what,
                (long long)c.layers, (long long)c.kv_heads);
  const int64_t eb = elem_bytes((int)c.dtype);
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || (c.layer_stride * eb) % 16 ||
      (c.page_stride * eb) % 16 || (c.head_stride * eb) % 16 || (c.slot_stride * eb) % 16 ||
      c.slot_stride < c.head_dim || c.head_stride < 0 || c.page_stride < 0 || c.layer_stride < 0)
    return fail(SSL_ERR_INVALID,
                "%s: the pools and their strides must be 16-byte aligned, positions at least "
                "head_dim apart", what);
  return SSL_OK;
}

namespace {

template <int DT>
struct Vec {
  static constexpr int VE = 16 / Elem<DT>::bytes;  // elements of a 16-byte vector
  __device__ __forceinline__ static void load(float* f, const void* base, int64_t off) {
    unpack16<DT>(f, *(const uint4*)((const char*)base + off * Elem<DT>::bytes));
  }
  __device__ __forceinline__ static void store(void* base, int64_t off, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == DT_F32) w[i] = __float_as_uint(f[i]);
      else w[i] = to_bits<DT>(f[2 * i]) | (to_bits<DT>(f[2 * i + 1]) << 16);
    }
    *(uint4*)((char*)base + off * Elem<DT>::bytes) = uint4{w[0], w[1], w[2], w[3]};
  }
};

// ---------------------------------------------------------------------------
// append: a row is one head of one token; LPR lanes hold it, each the VE
// features from j and their partners from j + HD / 2, so a rotation needs no
// exchange and a row's loads and stores are whole 16-byte vectors. Memory bounds
// it, below some hundred tokens the launch: 2048 tokens, 32 + 8 + 8 heads of 128
// with norms, bf16: 12.0 µs, 4.3 TB/s (a large copy here: 4.83); 16 tokens of 16
// heads: 4.0 µs.
// ---------------------------------------------------------------------------
struct AppendArgs {
  const char *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  const float *cos, *sin;
  int64_t cos_stride, sin_stride, angles;
  const void *q_norm, *k_norm;
  float eps;
  const int32_t *seq_ids, *positions;
  char* q_out;
  int64_t tokens;
  int heads;
};

template <int DT, int HD>
__global__ __launch_bounds__(256) void append_kernel(PagedCache C, AppendArgs A) {
  constexpr int VE = Vec<DT>::VE;
  constexpr int LPR = HD / 2 / VE;
  constexpr int RPW = 256 / LPR;  // rows a workgroup
  const int slots = A.heads + 2 * C.kv_heads;
  const int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / LPR;
  const int j = (threadIdx.x % LPR) * VE;
  const int64_t t = row / slots;
  if (t >= A.tokens) return;  // whole row groups leave together
  const int slot = (int)(row - t * slots);
  const int64_t pos = A.positions[t];
  const bool angle = pos >= 0 && pos < A.angles;
  const bool is_q = slot < A.heads, is_v = slot >= A.heads + C.kv_heads;
  const int head = is_q ? slot : (slot - A.heads) % C.kv_heads;
  int64_t dst = -1;  // elements from the pool's base
  if (is_q) {
    dst = (t * A.heads + head) * HD;
  } else {
    const int32_t s = A.seq_ids[t];
    const int64_t col = pos >> C.log2_page;
    if (angle && s >= 0 && s < C.seqs && col < C.cols) {
      const int32_t page = C.table[(int64_t)s * C.table_stride + col];
      if (C.has(page))
        dst = page * C.page_stride + head * C.head_stride + (pos & (C.page - 1)) * C.slot_stride;
    }
  }
  if (dst < 0) return;
  const void* src = is_q ? A.q : is_v ? A.v : A.k;
  const int64_t off = is_q ? t * A.q_token + head * A.q_head
                           : is_v ? t * A.v_token + head * A.v_head
                                  : t * A.k_token + head * A.k_head;
  float a[VE], b[VE];
  Vec<DT>::load(a, src, off + j);
  Vec<DT>::load(b, src, off + j + HD / 2);
  if (!is_v) {
    float c[VE], s[VE];
    const int64_t p = angle ? pos : 0;
#pragma unroll
    for (int e = 0; e < VE; e += 4) {
      const float4 cv = *(const float4*)(A.cos + p * A.cos_stride + j + e);
      const float4 sv = *(const float4*)(A.sin + p * A.sin_stride + j + e);
      c[e] = cv.x; c[e + 1] = cv.y; c[e + 2] = cv.z; c[e + 3] = cv.w;
      s[e] = sv.x; s[e + 1] = sv.y; s[e + 2] = sv.z; s[e + 3] = sv.w;
    }
    const void* norm = is_q ? A.q_norm : A.k_norm;
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor(ss, o);
      const float rs = rsqrtf(ss / (float)HD + A.eps);
      float w[VE];
      Vec<DT>::load(w, norm, j);
#pragma unroll
      for (int e = 0; e < VE; ++e) a[e] *= rs * w[e];
      Vec<DT>::load(w, norm, j + HD / 2);
#pragma unroll
      for (int e = 0; e < VE; ++e) b[e] *= rs * w[e];
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float x = a[e], y = b[e];
      a[e] = angle ? x * c[e] - y * s[e] : 0.f;
      b[e] = angle ? y * c[e] + x * s[e] : 0.f;
    }
  }
  void* out = is_q ? A.q_out : is_v ? C.v : C.k;
  Vec<DT>::store(out, dst + j, a);
  Vec<DT>::store(out, dst + j + HD / 2, b);
}

template <int DT>
void launch_append(const PagedCache& C, const AppendArgs& A, hipStream_t st) {
  const int64_t rows = A.tokens * (A.heads + 2 * C.kv_heads);
  const int rpw = 256 / (C.head_dim / 2 / Vec<DT>::VE);
  const dim3 grid((unsigned)((rows + rpw - 1) / rpw));
  if (C.head_dim == 64) hipLaunchKernelGGL((append_kernel<DT, 64>), grid, dim3(256), 0, st, C, A);
  else if (C.head_dim == 128)
    hipLaunchKernelGGL((append_kernel<DT, 128>), grid, dim3(256), 0, st, C, A);
  else hipLaunchKernelGGL((append_kernel<DT, 256>), grid, dim3(256), 0, st, C, A);
}

// ---------------------------------------------------------------------------
// Page operations
// ---------------------------------------------------------------------------
struct PagesArgs {
  const int32_t *lengths, *refs, *src, *dst;
  int n;
  int32_t *table_out, *lengths_out, *refs_out;
  uint8_t* ok;
  int32_t* live_out;
  int32_t* work;
};

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum of v over the workgroup's kPlanThreads threads; the sum
// in *total. Ends with a barrier, so the scratch may be used again at once.
__device__ __forceinline__ int scan_exclusive(int v, int* total) {
  __shared__ int part[kPlanThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) part[wave] = x;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) base += part[w];
    all += part[w];
  }
  __syncthreads();
  *total = all;
  return base + x - v;
}

__device__ __forceinline__ void copy_ints(int32_t* out, const int32_t* in, int64_t n, int64_t i0,
                                          int64_t step) {
  for (int64_t i = i0; i < n; i += step) out[i] = in[i];
}

// free, in one launch by one workgroup where the state is small: what each page
// loses is summed in shared memory, so no count is read back from memory, and a
// thread's loads all leave before it waits. Sixteen sequences of 4 entries: 2.7 µs
// in a graph, 4.4 as the two launches below; 32 of 64: 3.6, 4.4; with 8192 entries
// and as many pages 6.8, 4.5.
constexpr int kSmallState = 4096;  // entries, and pages
__global__ __launch_bounds__(kPlanThreads) void free_small_kernel(PagedCache C, PagesArgs A) {
  constexpr int kRounds = kSmallState / kPlanThreads;
  __shared__ uint8_t gone[kSmallState];  // a sequence has at least one entry
  __shared__ int lost[kSmallState];
  const int tid = threadIdx.x, entries = C.seqs * C.cols;
  int32_t page[kRounds], refs[kRounds], length[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int i = tid + k * kPlanThreads, s = i / C.cols;
    page[k] = i < entries ? C.table[(int64_t)s * C.table_stride + i - s * C.cols] : -1;
    refs[k] = i < C.pages ? A.refs[i] : 0;
    length[k] = i < C.seqs ? A.lengths[i] : 0;
    gone[i] = 0;
    lost[i] = 0;
  }
  __syncthreads();
  for (int i = tid; i < A.n; i += kPlanThreads) {
    const int s = A.dst[i];
    if (s >= 0 && s < C.seqs) gone[s] = 1;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int i = tid + k * kPlanThreads, s = i / C.cols;
    if (i < C.seqs) A.lengths_out[i] = gone[i] ? 0 : length[k];
    if (i >= entries) continue;
    A.table_out[i] = gone[s] ? -1 : page[k];
    if (gone[s] && C.has(page[k])) atomicAdd(&lost[page[k]], 1);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int p = tid + k * kPlanThreads;
    if (p < C.pages) A.refs_out[p] = refs[k] - lost[p];
  }
}

// free, launch 1: a workgroup per sequence writes its row and length (n_seq
// workgroups), the others copy the reference counts.
__global__ __launch_bounds__(256) void free_state_kernel(PagedCache C, PagesArgs A) {
  if ((int)blockIdx.x >= C.seqs) {
    copy_ints(A.refs_out, A.refs, C.pages,
              (int64_t)(blockIdx.x - C.seqs) * 256 + threadIdx.x,
              (int64_t)(gridDim.x - C.seqs) * 256);
    return;
  }
  const int s = blockIdx.x;
  int hit = 0;
  for (int i = threadIdx.x; i < A.n; i += 256) hit |= A.dst[i] == s;
  const bool gone = __syncthreads_or(hit);
  const int32_t* row = C.table + (int64_t)s * C.table_stride;
  int32_t* out = A.table_out + (int64_t)s * C.cols;
  for (int c = threadIdx.x; c < C.cols; c += 256) out[c] = gone ? -1 : row[c];
  if (threadIdx.x == 0) A.lengths_out[s] = gone ? 0 : A.lengths[s];
}

// free, launch 2: a workgroup per named sequence (the first to name it)
__global__ __launch_bounds__(256) void free_refs_kernel(PagedCache C, PagesArgs A) {
  const int i = blockIdx.x;
  const int s = A.dst[i];
  int hit = 0;
  for (int j = threadIdx.x; j < i; j += 256) hit |= A.dst[j] == s;
  if (__syncthreads_or(hit) || s < 0 || s >= C.seqs) return;
  const int32_t* row = C.table + (int64_t)s * C.table_stride;
  for (int c = threadIdx.x; c < C.cols; c += 256)
    if (C.has(row[c])) atomicAdd(&A.refs_out[row[c]], -1);
}

// fork, launch 1: workgroup 0 settles each fork (work[i]: the page its partly
// filled one is copied into, -1 where none is needed, -2 where it is refused);
// the others copy the state. kPlanThreads forks at a time: a wave checks a fork,
// its lanes the forks named before and the pages of the source; then the forks
// that need a page are ranked, and the lowest free pages, 4 a thread at a time.
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(PagedCache C, PagesArgs A) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int64_t i0 = (int64_t)(blockIdx.x - 1) * kPlanThreads + tid;
    const int64_t step = (int64_t)(gridDim.x - 1) * kPlanThreads;
    for (int64_t i = i0; i < (int64_t)C.seqs * C.cols; i += step)
      A.table_out[i] = C.table[i / C.cols * C.table_stride + i % C.cols];
    copy_ints(A.lengths_out, A.lengths, C.seqs, i0, step);
    copy_ints(A.refs_out, A.refs, C.pages, i0, step);
    return;
  }
  constexpr int kRefused = -2, kNone = -1, kNeeds = -3;
  __shared__ int state[kPlanThreads], fresh[kPlanThreads];
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the first pages' counts, on their way beside the forks' checks
  int first[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) first[k] = 4 * tid + k < C.pages ? A.refs[4 * tid + k] : 1;
  int taken = 0;  // free pages the forks before this run were given
  for (int base = 0; base < A.n; base += kPlanThreads) {
    const int count = min(A.n - base, kPlanThreads);
    for (int k = wave; k < count; k += kPlanThreads / 64) {
      const int s = A.src[base + k], d = A.dst[base + k];
      bool bad = s < 0 || s >= C.seqs || d < 0 || d >= C.seqs;
      int part = 0;
      if (!bad) {
        const int len = A.lengths[s];
        bad = A.lengths[d] != 0 || len < 0 || len > C.cols * C.page;
        const int pages = bad ? 0 : (len + C.page - 1) >> C.log2_page;
        for (int j = lane; j < base + k; j += 64) bad |= A.dst[j] == d;
        for (int c = lane; c < pages; c += 64)
          bad |= !C.has(C.table[(int64_t)s * C.table_stride + c]);
        part = len & (C.page - 1);
      }
      bad = __any(bad);
      if (lane == 0) state[k] = bad ? kRefused : part ? kNeeds : kNone;
    }
    __syncthreads();
    const int mine = tid < count ? state[tid] : kNone;
    int need;
    const int rank = scan_exclusive(mine == kNeeds, &need);
    int given = 0;  // free pages below the scan's place
    for (int64_t p0 = 0; p0 < C.pages && given < taken + need; p0 += 4 * kPlanThreads) {
      int idle[4], n_idle = 0;
      const int64_t p = p0 + 4 * tid;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        idle[k] = (p0 == 0 ? first[k] : p + k < C.pages ? A.refs[p + k] : 1) == 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) n_idle += idle[k];
      int total;
      int r = given + scan_exclusive(n_idle, &total) - taken;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (idle[k] && r >= 0 && r < need) fresh[r] = (int)(p + k);
        r += idle[k];
      }
      given += total;
    }
    __syncthreads();
    if (tid < count)
      A.work[base + tid] = mine != kNeeds ? mine : rank < given - taken ? fresh[rank] : kRefused;
    taken = min(given, taken + need);
    __syncthreads();
  }
}

// fork, launch 2: workgroup (x, fork): the fork's row, length and references (x = 0;
// pages that the ended sequence still held go back), and its share of the partly filled page's positions in every layer.
// 16 forks of sequences of up to 1500 positions, 16 layers of 16 heads of 128,
// bf16: 9.1 µs beside 5.4 of launch 1. (A wave a head instead of vectors over the
// device: the whole resampling 34 µs, this way 18.)
__global__ __launch_bounds__(256) void fork_copy_kernel(PagedCache C, PagesArgs A, int eb) {
  const int i = blockIdx.y;
  const int fresh = A.work[i];
  if (blockIdx.x == 0 && threadIdx.x == 0) A.ok[i] = fresh != -2;
  if (fresh == -2) return;
  const int s = A.src[i], d = A.dst[i];
  const int len = A.lengths[s];
  const int whole = len >> C.log2_page, part = len & (C.page - 1);
  const int32_t* row = C.table + (int64_t)s * C.table_stride;
  if (blockIdx.x == 0) {
    const int32_t* held = C.table + (int64_t)d * C.table_stride;
    int32_t* out = A.table_out + (int64_t)d * C.cols;
    for (int c = threadIdx.x; c < C.cols; c += 256) {
      if (C.has(held[c])) atomicAdd(&A.refs_out[held[c]], -1);
      const int32_t p = c < whole ? row[c] : (c == whole && part) ? fresh : -1;
      out[c] = p;
      if (p >= 0) atomicAdd(&A.refs_out[p], 1);
    }
    if (threadIdx.x == 0) A.lengths_out[d] = len;
  }
  if (!part) return;
  const int64_t from = row[whole] * C.page_stride, to = fresh * C.page_stride;
  const int log2_vec = __builtin_ctz(C.head_dim * eb / 16);  // 16-byte vectors a position
  const uint32_t per_head = (uint32_t)part << log2_vec;
  const uint32_t total = 2 * C.layers * C.kv_heads * per_head;  // below 2^31: the host checks
  for (uint32_t w = blockIdx.x * 256 + threadIdx.x; w < total; w += gridDim.x * 256) {
    const uint32_t head = w / per_head, x = w - head * per_head, l2 = head / C.kv_heads;
    const int64_t off = ((int64_t)(l2 >> 1) * C.layer_stride +
                         (int64_t)(head - l2 * C.kv_heads) * C.head_stride +
                         (int64_t)(x >> log2_vec) * C.slot_stride) * eb +
                        ((x & ((1 << log2_vec) - 1)) << 4);
    char* pool = (l2 & 1) ? C.v : C.k;
    *(uint4*)(pool + off + to * eb) = *(const uint4*)(pool + off + from * eb);
  }
}

// compact, launch 1 (one workgroup): L, the moves' (from, to) in work[0 .. 2L)
// behind the map work[2 pages .. 3 pages) of every page to its new number, and
// the new reference counts. A thread owns `seg` consecutive pages; u counts the
// pages in use below p, so a hole is the (p − u)-th and a page past L the
// (u − u(L))-th to move.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PagedCache C, PagesArgs A) {
  __shared__ int below;  // u(L)
  const int64_t P = C.pages;
  const int64_t seg = (P + kPlanThreads - 1) / kPlanThreads;
  const int64_t lo = min(threadIdx.x * seg, P), hi = min(lo + seg, P);
  int32_t *from = A.work, *to = A.work + P, *map = A.work + 2 * P;
  int used = 0, L;
  for (int64_t p = lo; p < hi; ++p) used += A.refs[p] > 0;
  const int before = scan_exclusive(used, &L);
  if (L == P && threadIdx.x == 0) below = L;
  if (lo <= L && L < hi) {
    int u = before;
    for (int64_t p = lo; p < L; ++p) u += A.refs[p] > 0;
    below = u;
  }
  __syncthreads();
  int u = before;
  for (int64_t p = lo; p < hi; ++p) {
    const int r = A.refs[p];
    const bool live = r > 0;
    map[p] = (int)p;
    A.refs_out[p] = p < L && live ? r : 0;
    if (!live && p < L) to[p - u] = (int)p;
    if (live && p >= L) from[u - below] = (int)p;
    u += live;
  }
  __syncthreads();
  const int total = L - below;
  for (int i = threadIdx.x; i < total; i += kPlanThreads) {
    map[from[i]] = to[i];
    A.refs_out[to[i]] = A.refs[from[i]];
  }
  if (threadIdx.x == 0) {
    *A.live_out = L;
    A.work[3 * P] = total;
  }
}

// compact, launch 2: the entries, and the moved pages' data, which bounds the
// call: 1024 moved pages of 8 layers, 8 heads of 128 and 16 positions, bf16: 218
// µs with launch 1's 8 over 4096 pages, 4.9 TB/s.
__global__ __launch_bounds__(256) void compact_copy_kernel(PagedCache C, PagesArgs A, int eb) {
  const int64_t P = C.pages;
  const int32_t *from = A.work, *to = A.work + P, *map = A.work + 2 * P;
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t i = i0; i < (int64_t)C.seqs * C.cols; i += step) {
    const int32_t p = C.table[i / C.cols * C.table_stride + i % C.cols];
    A.table_out[i] = C.has(p) ? map[p] : p;
  }
  const int moves = A.work[3 * P];
  const int log2_vec = __builtin_ctz(C.head_dim * eb / 16), log2_head = C.log2_page + log2_vec;
  const int heads = 2 * C.layers * C.kv_heads;
  for (int64_t w = i0; w < ((int64_t)moves * heads) << log2_head; w += step) {
    const uint32_t unit = (uint32_t)(w >> log2_head);  // move · heads + head
    const uint32_t i = unit / heads, head = unit - i * heads, l2 = head / C.kv_heads;
    const uint32_t x = (uint32_t)w & ((1u << log2_head) - 1);
    const int64_t off = ((int64_t)(l2 >> 1) * C.layer_stride +
                         (int64_t)(head - l2 * C.kv_heads) * C.head_stride +
                         (int64_t)(x >> log2_vec) * C.slot_stride) * eb +
                        ((x & ((1 << log2_vec) - 1)) << 4);
    char* pool = (l2 & 1) ? C.v : C.k;
    *(uint4*)(pool + off + to[i] * C.page_stride * eb) =
        *(const uint4*)(pool + off + from[i] * C.page_stride * eb);
  }
}

int pages_args(const char* what, const ssl_pages_args* a, bool pools, PagedCache* C, PagesArgs* A) {
  if (!a) return fail(SSL_ERR_INVALID, "%s: no arguments", what);
  if (int rc = paged_cache(what, a->cache, sizeof(ssl_pages_args), pools, C)) return rc;
  if (a->n < 0 || a->n > 65535)
    return fail(SSL_ERR_INVALID, "%s: %lld sequences", what, (long long)a->n);
  if (!a->refs || !a->refs_out || (C->seqs * (int64_t)C->cols > 0 && !a->table_out))
    return fail(SSL_ERR_INVALID, "%s: null pointer", what);
  *A = PagesArgs{a->lengths, a->refs, a->src, a->dst, (int)a->n, a->table_out, a->lengths_out,
                 a->refs_out, a->ok, a->live_out, (int32_t*)a->workspace};
  return SSL_OK;
}

unsigned blocks_for(int64_t items, int per, int64_t most) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + per - 1) / per, most));
}

}  // namespace
}  // namespace ssl

using namespace ssl;

extern "C" int ssl_paged_append(const ssl_paged_append_args* a, void* stream) {
  clear_error();
  const char* what = "paged_append";
  if (!a) return fail(SSL_ERR_INVALID, "%s: no arguments", what);
  PagedCache C;
  if (int rc = paged_cache(what, a->cache, sizeof(*a), true, &C)) return rc;
  if (a->tokens < 0 || a->heads <= 0 || a->heads > 65535 || a->angles < 0)
    return fail(SSL_ERR_INVALID, "%s: %lld tokens, %lld heads, %lld angles", what,
                (long long)a->tokens, (long long)a->heads, (long long)a->angles);
  if (a->tokens == 0) return SSL_OK;
  if (a->tokens * (a->heads + 2 * C.kv_heads) > 0x7fffffffLL * 8)
    return fail(SSL_ERR_UNSUPPORTED, "%s: %lld tokens in one call", what, (long long)a->tokens);
  if (!a->q || !a->k || !a->v || !a->cos || !a->sin || !a->seq_ids || !a->positions || !a->q_out ||
      a->angles == 0)
    return fail(SSL_ERR_INVALID, "%s: null pointer or no angles", what);
  const int64_t eb = elem_bytes((int)a->cache.dtype);
  for (int64_t s : {a->q_token, a->q_head, a->k_token, a->k_head, a->v_token, a->v_head})
    if ((s * eb) % 16) return fail(SSL_ERR_INVALID, "%s: rows must be 16-byte aligned", what);
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->cos, 16) ||
      !aligned(a->sin, 16) || !aligned(a->q_out, 16) || a->cos_stride % 4 || a->sin_stride % 4 ||
      (a->q_norm && !aligned(a->q_norm, 16)) || (a->k_norm && !aligned(a->k_norm, 16)))
    return fail(SSL_ERR_INVALID, "%s: q, k, v, the angles and the norms must be 16-byte aligned",
                what);
  AppendArgs A{(const char*)a->q, (const char*)a->k, (const char*)a->v, a->q_token, a->q_head,
               a->k_token, a->k_head, a->v_token, a->v_head, a->cos, a->sin, a->cos_stride,
               a->sin_stride, a->angles, a->q_norm, a->k_norm, (float)a->eps, a->seq_ids,
               a->positions, (char*)a->q_out, a->tokens, (int)a->heads};
  if (a->cache.dtype == SSL_F32) launch_append<DT_F32>(C, A, (hipStream_t)stream);
  else if (a->cache.dtype == SSL_BF16) launch_append<DT_BF16>(C, A, (hipStream_t)stream);
  else launch_append<DT_F16>(C, A, (hipStream_t)stream);
  return check_hip(hipGetLastError(), "paged_append launch");
}

extern "C" int ssl_pages_free(const ssl_pages_args* a, void* stream) {
  clear_error();
  PagedCache C;
  PagesArgs A;
  if (int rc = pages_args("pages_free", a, false, &C, &A)) return rc;
  if (C.seqs && (!A.lengths || !A.lengths_out || (A.n && !A.dst)))
    return fail(SSL_ERR_INVALID, "pages_free: null pointer");
  hipStream_t st = (hipStream_t)stream;
  if (C.cols > 0 && C.pages <= kSmallState && (int64_t)C.seqs * C.cols <= kSmallState) {
    hipLaunchKernelGGL(free_small_kernel, dim3(1), dim3(kPlanThreads), 0, st, C, A);
    return check_hip(hipGetLastError(), "pages_free launch");
  }
  hipLaunchKernelGGL(free_state_kernel, dim3(C.seqs + blocks_for(C.pages, 1024, 256)), dim3(256), 0,
                     st, C, A);
  if (A.n && C.seqs) hipLaunchKernelGGL(free_refs_kernel, dim3(A.n), dim3(256), 0, st, C, A);
  return check_hip(hipGetLastError(), "pages_free launch");
}

extern "C" int64_t ssl_pages_fork_workspace_size(int64_t n) { return n > 0 ? 4 * n : 0; }

extern "C" int ssl_pages_fork(const ssl_pages_args* a, void* stream) {
  clear_error();
  PagedCache C;
  PagesArgs A;
  if (int rc = pages_args("pages_fork", a, true, &C, &A)) return rc;
  if (C.seqs && (!A.lengths || !A.lengths_out))
    return fail(SSL_ERR_INVALID, "pages_fork: null pointer");
  if (A.n && (!A.src || !A.dst || !A.ok))
    return fail(SSL_ERR_INVALID, "pages_fork: null pointer");
  const int64_t need = ssl_pages_fork_workspace_size(A.n);
  if (A.n && (!A.work || a->workspace_bytes < need || !aligned(A.work, 4)))
    return fail(SSL_ERR_WORKSPACE, "pages_fork: workspace of %lld bytes needed", (long long)need);
  hipStream_t st = (hipStream_t)stream;
  const int eb = elem_bytes((int)a->cache.dtype);
  const int64_t state = std::max<int64_t>(C.pages, (int64_t)C.seqs * C.cols);
  const int64_t most = 2LL * C.layers * C.kv_heads * C.page * (C.head_dim * eb / 16);
  if (most > 0x7fffffff)
    return fail(SSL_ERR_UNSUPPORTED, "pages_fork: a page of all layers holds %lld bytes",
                (long long)most * 16);
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1 + blocks_for(state, kPlanThreads, 256)),
                     dim3(kPlanThreads), 0, st, C, A);
  if (A.n)
    hipLaunchKernelGGL(fork_copy_kernel, dim3(blocks_for(most, 1024, 4096), A.n), dim3(256), 0, st,
                       C, A, eb);
  return check_hip(hipGetLastError(), "pages_fork launch");
}

extern "C" int64_t ssl_pages_compact_workspace_size(int64_t pages) {
  return pages > 0 ? (3 * pages + 1) * 4 : 0;
}

extern "C" int ssl_pages_compact(const ssl_pages_args* a, void* stream) {
  clear_error();
  PagedCache C;
  PagesArgs A;
  if (int rc = pages_args("pages_compact", a, true, &C, &A)) return rc;
  if (!A.live_out) return fail(SSL_ERR_INVALID, "pages_compact: null pointer");
  const int64_t need = ssl_pages_compact_workspace_size(C.pages);
  if (!A.work || a->workspace_bytes < need || !aligned(A.work, 4))
    return fail(SSL_ERR_WORKSPACE, "pages_compact: workspace of %lld bytes needed",
                (long long)need);
  hipStream_t st = (hipStream_t)stream;
  const int eb = elem_bytes((int)a->cache.dtype);
  if (C.pages * 2 * C.layers * C.kv_heads > 0xffffffffLL)  // the copy numbers them in 32 bits
    return fail(SSL_ERR_UNSUPPORTED, "pages_compact: %lld pages of %d layers and %d heads",
                (long long)C.pages, C.layers, C.kv_heads);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, C, A);
  hipLaunchKernelGGL(compact_copy_kernel, dim3(2048), dim3(256), 0, st, C, A, eb);
  return check_hip(hipGetLastError(), "pages_compact launch");
}
