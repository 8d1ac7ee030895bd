// Attention over pages where a key/value head has few rows (query heads of its
// group times tokens): one new token per sequence, or a few.
//
// The keys and values are read once for 16 rows, so memory bounds it: per key
// 4·head_dim operations a row on 4·head_dim bytes (16-bit). Both products still
// run on the matrix cores, which take 16 rows at the cost of one, and keep the
// vector units free:
//
//   Sᵀ = K·Qᵀ   16 keys × 16 rows a tile. A lane's accumulators are 4 keys of
//               one row, so a row's maximum needs two exchanges.
//   Oᵀ = Vᵀ·Pᵀ  P as the accumulators leave it: a contraction may take the keys
//               in any order as long as V's lanes use the same, so neither
//               operand passes through LDS. A lane reads 16-byte pieces of the
//               8 (fp32: 4) keys it contracts and transposes them in registers.
//
// 16-bit products take a weight as two numbers of the type, itself rounded and what
// that left. Memory bounds the kernel, so the second product costs little (nothing of
// 88 µs at 60001 positions, 2 of 94 with a window of 1024, nothing of 15.8 at 16
// sequences of 1000), and outputs are as far from 64 bits as one rounding of the result
// makes them; with one number 5 to 9% farther.
//
// A wave takes every NW-th tile of its workgroup's part of the context and
// keeps its own running maximum, sum and output; the waves are joined through
// LDS, the parts of a split context by join_kernel: a second launch, 4 to 5 µs,
// which a counter in the workspace would save at the price of one that has to be
// kept at zero between calls.
//
// Measured: contexts of up to 60001 positions of 4 sequences, 32 heads over 8 of
// 128, bf16: 88 µs, 4.86 TB/s (a large copy here: 4.83); 64 sequences, a window of
// 1024, 16 heads: 96 µs, 4.65 TB/s. One sequence of 717, 16 heads of 64: 7.8 µs, the
// latency of a launch, of the table, of three loads in turn and of the join of waves.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "paged_join.h"

namespace ssl {
namespace {

constexpr int kRows = 16;  // rows a workgroup takes

template <int DT, int HD>
struct Shape {
  static constexpr int EB = Elem<DT>::bytes;
  static constexpr int NS = DT == DT_F32 ? 1 : 2;  // 16-key subtiles a tile
  static constexpr int T = 16 * NS;
  static constexpr int KE = DT == DT_F32 ? 4 : 8;
  static constexpr int KS = HD / (4 * KE);  // contraction steps of Sᵀ
  // values: a lane's vectors of VE features, U of them a key
  static constexpr int VE = std::min(HD / 16, 16 / EB);
  static constexpr int U = HD / 16 / VE;
  static constexpr int VD = VE * EB / 4;  // dwords of a vector
};

// Waves of a wide workgroup: as many as its registers allow at once.
constexpr int wide_waves(int dt, int hd) {
  return hd == 64 ? 16 : dt == DT_F32 && hd == 256 ? 4 : 8;
}

// Rows of a sequence and key/value head at most (tokens of one sequence).
int64_t max_rows(const AttnArgs& A, int G) { return A.cu ? A.tokens * G : G; }

// VD dwords from a 4·VD-byte aligned address
template <int VD>
__device__ __forceinline__ void load_dwords(uint32_t* r, const char* p) {
  if constexpr (VD == 4) {
    const uint4 v = *(const uint4*)p;
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else {
    const uint2 v = *(const uint2*)p;
    r[0] = v.x; r[1] = v.y;
  }
}

// CHUNKS: tokens by cu, each row with a position of its own; else one token a
// sequence, whose position is a scalar.
template <int DT, int HD, int NW, bool CHUNKS>
__global__ __launch_bounds__(NW * 64, NW > 4 ? NW / 4 : DT == DT_F32 && HD == 256 ? 1 : 2)
void decode_kernel(PagedCache C, AttnArgs A, int n_blocks) {
  using S = Shape<DT, HD>;
  using M = Mma<DT, S::KE>;
  using Frag = typename M::Frag;
  extern __shared__ float sh_o[];  // [NW][rows][HD]
  __shared__ float sh_m[NW][kRows], sh_l[NW][kRows];
  __shared__ uint32_t sh_anew;  // rows to be taken anew

  const int G = A.heads / C.kv_heads;
  const int kh = blockIdx.y / n_blocks;
  const int s = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  if (CHUNKS && s == C.seqs) {
    if (blockIdx.x == 0 && blockIdx.y % n_blocks == 0)
      zero_tail(C, A, kh, HD * S::EB / 16, threadIdx.x, NW * 64);
    return;
  }
  const Chunk chunk = CHUNKS ? Chunk(C, A, s, G) : Chunk(C, A, s);
  const int n_rows = CHUNKS ? chunk.rows : G;
  for (int block = blockIdx.y % n_blocks; block * kRows < n_rows; block += n_blocks) {
    const int row_a = block * kRows, rows = min(n_rows - row_a, kRows);
    // row c and its position; the block's range of them
    const int r = row_a + min(c, rows - 1);
    const int64_t token = CHUNKS ? chunk.t0 + r / G : s;
    const int head = kh * G + (CHUNKS ? r % G : r);
    const int p_min = CHUNKS ? chunk.p0 + row_a / G : chunk.p0;
    const int p_max = CHUNKS ? chunk.p0 + (row_a + rows - 1) / G : p_min;
    const int p = CHUNKS ? chunk.p0 + r / G : p_min;
    const auto first_of = [&](int q) {
      return A.window && q + 1 > A.window ? q + 1 - A.window : 0;
    };
    const int first = first_of(p), first_min = first_of(p_min), first_max = first_of(p_max);
    const TileRange range = tile_range<S::T>(max(p_min, 0), p_max, A.window, A.sinks);
    const int per = part_tiles(A, range.count);
    const int lo = blockIdx.x * per, hi = min(lo + per, range.count);
    const bool whole = per >= range.count;
    if (lo >= hi && blockIdx.x > 0) continue;  // the join reads no part past the last

    Frag qf[S::KS];
  #pragma unroll
    for (int i = 0; i < S::KS; ++i)
      qf[i] = load_kfrag<DT, S::KE>(
          A.q, token * A.q_token + (int64_t)head * A.q_head + (4 * i + g) * S::KE, S::KE);

    {
      uint32_t* q = (uint32_t*)qf;
      const uint32_t flip = A.flip & (DT == DT_F32 ? 0x80000000u : 0x80008000u);
  #pragma unroll
      for (int i = 0; i < (int)(sizeof qf / 4); ++i) q[i] = (q[i] & A.keep) ^ flip;
    }

    // lane offsets within a page's head: key c for K, keys 4g + e for V
    const uint32_t slot_bytes = (uint32_t)(C.slot_stride * S::EB);
    const uint32_t k_off = c * slot_bytes + g * S::KE * S::EB;
    const uint32_t v_off = 4 * g * slot_bytes + c * S::VE * S::EB;
    const int64_t head_off = kh * C.head_stride;
    const int32_t* row = C.table + (int64_t)s * C.table_stride;

    f32x4 o[S::U * S::VE];
  #pragma unroll
    for (int i = 0; i < S::U * S::VE; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // of head c; l: this lane's keys only
    // fp16 weights are kept 256-fold, so that small ones keep their digits
    constexpr float kBias = DT == DT_F16 ? 8.f : 0.f;

    // pages of the wave's next tile, read a tile ahead
    int32_t page[S::NS];
    auto pages_of = [&](int i, int32_t* pg) {
      const int key0 = range.tile(min(i, hi - 1)) * S::T;
  #pragma unroll
      for (int t = 0; t < S::NS; ++t)
        pg[t] = row[min((key0 + 16 * t) >> C.log2_page, C.cols - 1)];
    };
    if (lo + wave < hi) pages_of(lo + wave, page);

    for (int i = lo + wave; i < hi; i += NW) {
      const int key0 = range.tile(i) * S::T;
      const char *kb[S::NS], *vb[S::NS];
      bool all = key0 + S::T - 1 <= p_min && (key0 >= first_max || key0 + S::T <= A.sinks);
      bool has[S::NS];
  #pragma unroll
      for (int t = 0; t < S::NS; ++t) {
        has[t] = C.has(page[t]);
        all = all && has[t];
        const int64_t off = ((has[t] ? page[t] : 0) * C.page_stride + head_off +
                             ((key0 + 16 * t) & (C.page - 1)) * C.slot_stride) * S::EB;
        kb[t] = C.k + off;
        vb[t] = C.v + off;
      }
      Frag kf[S::NS][S::KS];
      uint32_t vr[S::NS][4][S::U][S::VD];
  #pragma unroll
      for (int t = 0; t < S::NS; ++t)
  #pragma unroll
        for (int k = 0; k < S::KS; ++k)
          kf[t][k] = load_kfrag_full<DT, S::KE>(kb[t] + k_off + k * 4 * S::KE * S::EB, 0);
  #pragma unroll
      for (int t = 0; t < S::NS; ++t)
  #pragma unroll
        for (int e = 0; e < 4; ++e)
  #pragma unroll
          for (int w = 0; w < S::U; ++w)
            load_dwords<S::VD>(vr[t][e][w], vb[t] + (size_t)(e * slot_bytes) + v_off +
                                                w * 16 * S::VE * S::EB);
      if (i + NW < hi) pages_of(i + NW, page);
      __builtin_amdgcn_sched_barrier(0);

      f32x4 acc[S::NS];
  #pragma unroll
      for (int t = 0; t < S::NS; ++t) {
        acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  #pragma unroll
        for (int k = 0; k < S::KS; ++k) M::run(acc[t], kf[t][k], qf[k]);
      }
      float x[S::NS][4];
  #pragma unroll
      for (int t = 0; t < S::NS; ++t)
  #pragma unroll
        for (int e = 0; e < 4; ++e) x[t][e] = rounded(acc[t][e] * A.scale_log2);
      if (!all) {  // what a row does not see: no weight; what none sees may hold anything
  #pragma unroll
        for (int t = 0; t < S::NS; ++t)
  #pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * t + 4 * g + e;
            const bool mine = has[t] && key <= p && (key >= first || key < A.sinks);
            const bool see = has[t] && key <= p_max && (key >= first_min || key < A.sinks);
            x[t][e] = mine ? x[t][e] : -INFINITY;
  #pragma unroll
            for (int w = 0; w < S::U; ++w)
  #pragma unroll
              for (int d = 0; d < S::VD; ++d) vr[t][e][w][d] = see ? vr[t][e][w][d] : 0u;
          }
      }
      float mx = m;
  #pragma unroll
      for (int t = 0; t < S::NS; ++t)
  #pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, x[t][e]);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float base = mx == -INFINITY ? 0.f : mx;
      if (__any(mx > m)) {
        const float a = exp2f(m - base);
        l *= a;
  #pragma unroll
        for (int k = 0; k < S::U * S::VE; ++k) o[k] *= a;
      }
      m = mx;
  #pragma unroll
      for (int t = 0; t < S::NS; ++t)
  #pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[t][e] = __builtin_amdgcn_exp2f(kBias ? x[t][e] - base + kBias : x[t][e] - base);
          l += x[t][e];
        }
      Frag pf, pl;  // the weights; what their rounding left
      if constexpr (DT == DT_F32) {
  #pragma unroll
        for (int e = 0; e < 4; ++e) pf.f[e] = x[0][e];
      } else {
  #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = x[i / 2][2 * (i % 2)], b = x[i / 2][2 * (i % 2) + 1];
          pf.d[i] = pack2<DT>(a, b);
          pl.d[i] = pack2<DT>(a - low16<DT>(pf.d[i]), b - low16<DT>(pf.d[i] >> 16));
        }
      }
  #pragma unroll
      for (int w = 0; w < S::U; ++w)
  #pragma unroll
        for (int f = 0; f < S::VE; ++f) {
          Frag vf;
          if constexpr (DT == DT_F32) {
  #pragma unroll
            for (int e = 0; e < 4; ++e) vf.f[e] = __uint_as_float(vr[0][e][w][f]);
          } else {
  #pragma unroll
            for (int d = 0; d < 4; ++d) {
              const uint32_t a = vr[d / 2][2 * (d % 2)][w][f / 2];
              const uint32_t b = vr[d / 2][2 * (d % 2) + 1][w][f / 2];
              vf.d[d] = __builtin_amdgcn_perm(b, a, f % 2 ? 0x07060302u : 0x05040100u);
            }
          }
          M::run(o[w * S::VE + f], vf, pf);
          if constexpr (DT != DT_F32) M::run(o[w * S::VE + f], vf, pl);
        }
    }

    // join the waves: sums over the lane groups, then o through LDS
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
      sh_m[wave][c] = m;
      sh_l[wave][c] = l;
    }
    if (c < rows) {
  #pragma unroll
      for (int w = 0; w < S::U; ++w)
  #pragma unroll
        for (int e = 0; e < 4; ++e) {
          float* to = sh_o + (wave * rows + c) * HD + w * 16 * S::VE + (4 * g + e) * S::VE;
  #pragma unroll
          for (int f = 0; f < S::VE; f += 4)
            *(f32x4*)(to + f) = f32x4{o[w * S::VE + f][e], o[w * S::VE + f + 1][e],
                                      o[w * S::VE + f + 2][e], o[w * S::VE + f + 3][e]};
        }
    }
    if (CHUNKS && threadIdx.x == 0) sh_anew = 0;
    __syncthreads();
    for (int i = threadIdx.x * 4; i < rows * HD; i += NW * 256) {
      const int k = i / HD, d = i % HD;
      float top = sh_m[0][k];
  #pragma unroll
      for (int w = 1; w < NW; ++w) top = fmaxf(top, sh_m[w][k]);
      const float base = top == -INFINITY ? 0.f : top;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
  #pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float a = exp2f(sh_m[w][k] - base);
        sum += sh_l[w][k] * a;
        acc += *(const f32x4*)(sh_o + (w * rows + k) * HD + d) * a;
      }
      // (a row whose sum is NaN is NaN by its own scores)
      if (CHUNKS && sum == sum &&
          !(acc[0] * 0.f + acc[1] * 0.f + acc[2] * 0.f + acc[3] * 0.f == 0.f))
        atomicOr(&sh_anew, 1u << k);
      const int64_t at = CHUNKS
                             ? (chunk.t0 + (row_a + k) / G) * A.heads + kh * G + (row_a + k) % G
                             : (int64_t)s * A.heads + kh * G + row_a + k;
      if (whole) {
        acc *= sum == 0.f ? 0.f : 1.f / sum;
        if constexpr (DT == DT_F32)
          *(f32x4*)(A.out + (at * HD + d) * 4) = acc;
        else
          *(uint2*)(A.out + (at * HD + d) * 2) =
              uint2{pack2<DT>(acc[0], acc[1]), pack2<DT>(acc[2], acc[3])};
      } else {
        *(f32x4*)(A.part_o + ((at * A.n_split + blockIdx.x) * HD + d)) = acc;
        if (d == 0) {
          float* ml = A.part_ml + 2 * (at * A.n_split + blockIdx.x);
          ml[0] = top;
          ml[1] = sum;
        }
      }
    }
    if (!CHUNKS) return;  // n_blocks covers the group, whose rows see the same
    __syncthreads();
    const uint32_t anew = __builtin_amdgcn_readfirstlane(sh_anew);
    for (int k = anew ? wave : rows; k < rows; k += NW) {
      if (!(anew >> k & 1)) continue;
      float top = sh_m[0][k], sum = 0.f;
#pragma unroll
      for (int w = 1; w < NW; ++w) top = fmaxf(top, sh_m[w][k]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < NW; ++w) sum += sh_l[w][k] * exp2f(sh_m[w][k] - base);
      const int rk = row_a + k;
      const int64_t tk = chunk.t0 + rk / G;
      const int hk = kh * G + rk % G;
      row_anew<DT, HD, S::T>(
          C, A, s, kh, tk, hk, chunk.p0 + rk / G, range, lo, hi, sum,
          whole ? nullptr : A.part_o + ((tk * A.heads + hk) * A.n_split + blockIdx.x) * HD,
          [](int) { return true; });
    }
    if ((block + n_blocks) * kRows >= n_rows) return;
    __syncthreads();  // the next rows use the same LDS
  }
}

template <int DT, int HD, int NW, bool CHUNKS>
int launch_waves(const PagedCache& C, const AttnArgs& A, int64_t max_tokens, hipStream_t st) {
  const int G = A.heads / C.kv_heads;
  const int n_blocks = (int)std::max<int64_t>(1, (max_tokens * G + kRows - 1) / kRows);
  const size_t lds = NW * sizeof(float) * HD * std::min<int64_t>(max_rows(A, G), kRows);
  if (lds + 4096 > 64 * 1024) {  // beside the static arrays
    static std::atomic<uint64_t> raised{0};
    if (int rc = allow_lds((const void*)decode_kernel<DT, HD, NW, CHUNKS>,
                           NW * (int)sizeof(float) * HD * kRows, &raised))
      return rc;
  }
  const dim3 grid((unsigned)A.n_split, (unsigned)(C.kv_heads * n_blocks),
                  (unsigned)(C.seqs + (A.cu ? 1 : 0)));
  hipLaunchKernelGGL((decode_kernel<DT, HD, NW, CHUNKS>), grid, dim3(NW * 64), lds, st, C, A,
                     n_blocks);
  if (A.n_split > 1) launch_join<DT, HD, Shape<DT, HD>::T, kRows>(C, A, st);
  return SSL_OK;
}

template <int DT, int HD>
int launch(const PagedCache& C, const AttnArgs& A, int64_t max_tokens, hipStream_t st) {
  constexpr int WIDE = wide_waves(DT, HD);
  if (A.cu)
    return A.waves == 4 ? launch_waves<DT, HD, 4, true>(C, A, max_tokens, st)
                        : launch_waves<DT, HD, WIDE, true>(C, A, max_tokens, st);
  return A.waves == 4 ? launch_waves<DT, HD, 4, false>(C, A, max_tokens, st)
                      : launch_waves<DT, HD, WIDE, false>(C, A, max_tokens, st);
}

template <int DT>
int launch_dt(const PagedCache& C, const AttnArgs& A, int64_t max_tokens, hipStream_t st) {
  if (C.head_dim == 64) return launch<DT, 64>(C, A, max_tokens, st);
  if (C.head_dim == 128) return launch<DT, 128>(C, A, max_tokens, st);
  return launch<DT, 256>(C, A, max_tokens, st);
}

}  // namespace

// One part where a wide workgroup's waves take the longest context in 3 steps,
// or in 6 where there are workgroups enough to keep the device busy meanwhile (16
// sequences of 1000 positions, 16 heads of 128: 16 µs, in 8 parts of narrow ones
// 20; 64 of 300, 8 key/value heads: 11 and 15); else parts of about 1/2048 of
// the longest possible work, of 4 tiles (one a wave) at least. The estimate: 6 µs
// and every 16 rows' reading of their context at 7 TB/s, the rate from the caches
// (2.7 for 256-wide heads, whose registers leave room for half the waves), or
// their products at 80 TFLOP/s in fp32.
int64_t paged_decode_plan(const PagedCache& C, AttnArgs* A, int dtype, int64_t max_tokens,
                          int64_t max_length) {
  const int T = dtype == SSL_F32 ? 16 : 32;
  const int G = A->heads / C.kv_heads;
  const int64_t blocks = C.seqs * std::max<int64_t>(1, (max_tokens * G + kRows - 1) / kRows) *
                         C.kv_heads;
  int64_t reach = max_length;
  if (A->window)
    reach = std::min<int64_t>(reach, (int64_t)A->window + std::min(A->sinks, 0x3fffffff) +
                                         (max_tokens > 1 ? kRows : 0) + 2 * T);
  const int64_t tiles = std::max<int64_t>(1, (reach + T - 1) / T);
  const int64_t rows16 = std::min<int64_t>(blocks, C.kv_heads * (A->tokens * G / kRows + C.seqs));
  const double read = (double)rows16 * C.head_dim *
                      std::min<int64_t>(reach, std::max<int64_t>(max_length - max_tokens / 2, 1));
  A->us = (float)(6 + std::max(read * 2 * elem_bytes(dtype) / (C.head_dim == 256 ? 2.7e6 : 7e6),
                               dtype == SSL_F32 ? read * 4 * kRows / 80e6 : 0.));
  const int wide = wide_waves(dtype, C.head_dim);
  A->n_split = 1;
  A->per = (int)std::min<int64_t>(tiles, 0x3fffffff);
  A->waves = 4;
  if (tiles <= 4) return 0;
  const int64_t steps = (tiles + wide - 1) / wide;
  if (wide > 4 && blocks * wide <= 4096 && (steps <= 3 || (steps <= 6 && blocks >= 128))) {
    A->waves = wide;
    return 0;
  }
  int64_t per = std::max<int64_t>(4, (tiles * blocks + 2047) / 2048);
  per = (per + 3) / 4 * 4;
  A->per = (int)std::min<int64_t>(per, 0x3fffffff);
  A->n_split = (int)std::min<int64_t>((tiles + per - 1) / per, 65535);
  if (A->n_split <= 1) return 0;
  return A->tokens * A->heads * (int64_t)A->n_split * (C.head_dim + 2) * 4;
}

int paged_decode_launch(const PagedCache& C, const AttnArgs& A, int dtype, int64_t max_tokens,
                        hipStream_t st) {
  int rc;
  if (dtype == SSL_F32) rc = launch_dt<DT_F32>(C, A, max_tokens, st);
  else if (dtype == SSL_BF16) rc = launch_dt<DT_BF16>(C, A, max_tokens, st);
  else rc = launch_dt<DT_F16>(C, A, max_tokens, st);
  return rc ? rc : check_hip(hipGetLastError(), "paged attention launch");
}

}  // namespace ssl
