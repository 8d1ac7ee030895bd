// What the two attention kernels share: rows taken anew, and the parts of split
// contexts joined: a row's parts hold their maximum m, sum l and output o relative
// to m; the row is Σ o·2^(m − max) / Σ l·2^(m − max).
#pragma once

#include "paged.h"

namespace ssl {

// Row `at` (token · heads + head) of a call whose workgroups took ROWS packed
// rows and tiles of T positions: its sequence's chunk, or false for none.
template <int T, int ROWS>
__device__ __forceinline__ int row_parts(const PagedCache& C, const AttnArgs& A, int64_t at) {
  const int64_t t = at / A.heads;
  int a = (int)t;
  if (A.cu) {
    a = 0;
    int b = C.seqs;  // the first sequence whose end lies past t
    while (a < b) {
      const int mid = (a + b) >> 1;
      if (A.cu[mid + 1] > t) b = mid;
      else a = mid + 1;
    }
    if (a >= C.seqs) return 0;
  }
  const int G = A.heads / C.kv_heads;
  const Chunk chunk(C, A, a, G);
  const int r = (int)(t - chunk.t0) * G + (int)(at % A.heads) % G;
  if (r < 0 || r >= chunk.rows) return 0;
  const int row_a = r / ROWS * ROWS, row_b = min(row_a + ROWS, chunk.rows) - 1;
  const TileRange range = tile_range<T>(max(chunk.p0 + row_a / G, 0), chunk.p0 + row_b / G,
                                        A.window, A.sinks);
  const int per = part_tiles(A, range.count);
  return per >= range.count ? 0 : (range.count + per - 1) / per;  // one part wrote the output
}

// The tiles' products give a masked position the weight 0, which takes a NaN or an
// infinity among its values into the row all the same. A row whose output is not
// finite is therefore taken anew over tiles lo … hi − 1, by a wave, from the
// positions that it sees alone: their average, which a part holds times its sum `l`
// (scores of masked positions never entered that). (600 tokens of 2 heads of 128, all
// values NaN: 680 µs, finite 24; 4096 tokens of 16 heads 23 ms, 92 µs.)
// part: where the row's part goes, or null for the output; mine(f): the features to
// write.
template <int DT, int HD, int T, typename F>
__device__ __forceinline__ void row_anew(const PagedCache& C, const AttnArgs& A, int s, int kh,
                                         int64_t token, int head, int p, const TileRange& range,
                                         int lo, int hi, float l, float* part, F mine) {
  constexpr int N = HD / 64, EB = Elem<DT>::bytes;
  const int lane = threadIdx.x & 63, f0 = lane * N;
  const char* q = A.q + (token * A.q_token + (int64_t)head * A.q_head) * EB;
  const int32_t* row = C.table + (int64_t)s * C.table_stride;
  const int first = A.window && p + 1 > A.window ? p + 1 - A.window : 0;
  const float sign = A.flip ? -A.scale_log2 : A.scale_log2;
  float o[N], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  for (int i = lo; i < hi; ++i) {
    // scores: a lane a position
    const int key = range.tile(i) * T + lane;
    bool see = lane < T && key <= p && (key >= first || key < A.sinks);
    const int32_t page = see ? row[min(key >> C.log2_page, C.cols - 1)] : -1;
    see = see && C.has(page);
    const int64_t off = (see ? page * C.page_stride + (key & (C.page - 1)) * C.slot_stride : 0) +
                        kh * C.head_stride;
    float x = 0.f;
#pragma unroll 1  // the kernels' registers are for their own loops
    for (int j = 0; j < HD; j += 16 / EB) {
      const uint4 a = *(const uint4*)(q + j * EB), b = *(const uint4*)(C.k + (off + j) * EB);
#pragma unroll
      for (int e = 0; e < 16 / EB; ++e)
        x = fmaf(A.keep ? load_scalar<DT>(&a, e) : 0.f, load_scalar<DT>(&b, e), x);
    }
    x = see ? rounded(x * sign) : -INFINITY;
    float top = fmaxf(m, x);
#pragma unroll
    for (int b = 1; b < 64; b <<= 1) top = fmaxf(top, __shfl_xor(top, b));
    const float base = top == -INFINITY ? 0.f : top, a = exp2f(m - base);
    const float w = exp2f(x - base);
    m = top;
    sum = fmaf(sum, a, w);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] *= a;
    // values: a lane N features; a position not seen reads page 0 and counts as zero
    const uint64_t seen = __ballot(see);
    if (!seen) continue;
#pragma unroll 4
    for (int c = 0; c < T; ++c) {
      const float wc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), c));
      const int64_t at = ((int64_t)__builtin_amdgcn_readlane((int)(off >> 32), c) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)off, c);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float v = load_scalar<DT>(C.v, at + f0 + j);
        o[j] = fmaf(wc, seen >> c & 1 ? v : 0.f, o[j]);
      }
    }
  }
#pragma unroll
  for (int b = 1; b < 64; b <<= 1) sum += __shfl_xor(sum, b);
  const float by = sum == 0.f ? 0.f : (part ? l : 1.f) / sum;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int f = f0 + i;
    if (!mine(f)) continue;
    const int64_t at = (token * A.heads + head) * HD + f;
    if (part) part[f] = o[i] * by;
    else if constexpr (DT == DT_F32) ((float*)A.out)[at] = o[i] * by;
    else ((uint16_t*)A.out)[at] = (uint16_t)to_bits<DT>(o[i] * by);
  }
}

// TPR threads a row: HD / 4 lanes take the features, the lane groups every
// (4 TPR / HD)-th part. A wave a row for many rows, a workgroup a row for few
// (whose parts are many).
template <int DT, int HD, int T, int ROWS, int TPR>
__global__ __launch_bounds__(256) void join_kernel(PagedCache C, AttnArgs A) {
  constexpr int LN = HD / 4, NG = TPR / LN;
  __shared__ f32x4 sh_o[TPR == 256 ? NG : 1][LN];
  __shared__ float sh_l[NG];
  const int64_t at = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (at >= A.tokens * A.heads) return;
  const int parts = row_parts<T, ROWS>(C, A, at);
  if (parts == 0) return;
  const int lane = threadIdx.x & 63;
  const int d = threadIdx.x % LN, grp = threadIdx.x % TPR / LN;
  const float* ml = A.part_ml + 2 * at * A.n_split;
  const float* po = A.part_o + at * A.n_split * HD + 4 * d;
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 64) top = fmaxf(top, ml[2 * i]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int i = grp; i < parts; i += NG) {
    const float x = exp2f(ml[2 * i] - base);
    sum += ml[2 * i + 1] * x;
    acc += *(const f32x4*)(po + (int64_t)i * HD) * x;
  }
  if constexpr (TPR == 256) {
    sh_o[grp][d] = acc;
    if (d == 0) sh_l[grp] = sum;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int i = 1; i < NG; ++i) {
      acc += sh_o[i][d];
      sum += sh_l[i];
    }
  } else {
#pragma unroll
    for (int o = LN; o < 64; o <<= 1) {
      sum += __shfl_xor(sum, o);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
    }
    if (grp) return;
  }
  acc *= sum == 0.f ? 0.f : 1.f / sum;
  if constexpr (DT == DT_F32)
    *(f32x4*)(A.out + (at * HD + 4 * d) * 4) = acc;
  else
    *(uint2*)(A.out + (at * HD + 4 * d) * 2) =
        uint2{pack2<DT>(acc[0], acc[1]), pack2<DT>(acc[2], acc[3])};
}

template <int DT, int HD, int T, int ROWS>
void launch_join(const PagedCache& C, const AttnArgs& A, hipStream_t st) {
  const int64_t rows = A.tokens * A.heads;
  if (rows <= 2048)
    hipLaunchKernelGGL((join_kernel<DT, HD, T, ROWS, 256>), dim3((unsigned)rows), dim3(256), 0, st,
                       C, A);
  else
    hipLaunchKernelGGL((join_kernel<DT, HD, T, ROWS, 64>), dim3((unsigned)((rows + 3) / 4)),
                       dim3(256), 0, st, C, A);
}

}  // namespace ssl
