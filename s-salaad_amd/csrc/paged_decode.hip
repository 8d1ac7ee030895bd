// Attention of one new token per sequence over its pages.
//
// The keys and values are read once, so memory bounds it: per key 4·head_dim
// operations a query head on 4·head_dim bytes (16-bit, one head per key/value
// head). Both products still run on the matrix cores, which take a group of up
// to 16 query heads at the cost of one, and keep the vector units free:
//
//   Sᵀ = K·Qᵀ   16 keys × 16 heads a tile. A lane's accumulators are 4 keys of
//               one head, so a head's maximum needs two exchanges.
//   Oᵀ = Vᵀ·Pᵀ  P as the accumulators leave it: a contraction may take the keys
//               in any order as long as V's lanes use the same, so neither
//               operand passes through LDS. A lane reads 16-byte pieces of the
//               8 (fp32: 4) keys it contracts and transposes them in registers.
//
// A wave takes every fourth tile of its workgroup's part of the context and
// keeps its own running maximum, sum and output; the waves are joined through
// LDS, the parts of a split context by join_kernel.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "paged.h"

namespace ssl {
namespace {

constexpr int kHeadRows = 16;  // query heads a workgroup takes at most

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

template <int DT, int HD>
__global__ __launch_bounds__(256, DT == DT_F32 && HD == 256 ? 1 : 2) void decode_kernel(PagedCache C, AttnArgs A) {
  using S = Shape<DT, HD>;
  using M = Mma<DT, S::KE>;
  using Frag = typename M::Frag;
  extern __shared__ float sh_o[];  // [4][rows][HD]
  __shared__ float sh_m[4][kHeadRows], sh_l[4][kHeadRows];

  const int G = A.heads / C.kv_heads;
  const int n_hb = (G + kHeadRows - 1) / kHeadRows;
  const int kh = blockIdx.y / n_hb, g0 = (blockIdx.y % n_hb) * kHeadRows;
  const int rows = min(G - g0, kHeadRows), h0 = kh * G + g0;
  const int64_t s = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;

  const int p = min(A.lengths[s], C.cols << C.log2_page) - 1;
  const int first = A.window && p + 1 > A.window ? p + 1 - A.window : 0;
  const TileRange range = tile_range<S::T>(p, p, A.window, A.sinks);
  const int per = part_tiles(A, range.count);
  const int lo = blockIdx.x * per, hi = min(lo + per, range.count);
  const bool whole = per >= range.count;
  if (lo >= hi && blockIdx.x > 0) return;  // the join reads no part past the last

  Frag qf[S::KS];
#pragma unroll
  for (int i = 0; i < S::KS; ++i)
    qf[i] = load_kfrag<DT, S::KE>(
        A.q, s * A.q_token + (int64_t)(h0 + min(c, rows - 1)) * A.q_head + (4 * i + g) * S::KE,
        S::KE);

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
  const int32_t* row = C.table + s * C.table_stride;

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

  for (int i = lo + wave; i < hi; i += 4) {
    const int key0 = range.tile(i) * S::T;
    const char *kb[S::NS], *vb[S::NS];
    bool all = key0 + S::T - 1 <= p && (key0 >= first || key0 + S::T <= A.sinks);
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
          load_dwords<S::VD>(vr[t][e][w], vb[t] + (size_t)(e * slot_bytes) + v_off + w * 16 * S::VE * S::EB);
    if (i + 4 < hi) pages_of(i + 4, page);
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
      for (int e = 0; e < 4; ++e) x[t][e] = acc[t][e] * A.scale_log2;
    if (!all) {  // what is not seen: no weight, and values that may hold anything
#pragma unroll
      for (int t = 0; t < S::NS; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 16 * t + 4 * g + e;
          const bool see = has[t] && key <= p && (key >= first || key < A.sinks);
          x[t][e] = see ? x[t][e] : -INFINITY;
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
    const float base = (mx == -INFINITY ? 0.f : mx) - kBias;
    if (__any(mx > m)) {
      const float a = exp2f(m - (base + kBias));
      l *= a;
#pragma unroll
      for (int k = 0; k < S::U * S::VE; ++k) o[k] *= a;
    }
    m = mx;
#pragma unroll
    for (int t = 0; t < S::NS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[t][e] = exp2f(x[t][e] - base);
        l += x[t][e];
      }
    Frag pf;
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) pf.f[e] = x[0][e];
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        pf.d[2 * t] = pack2<DT>(x[t][0], x[t][1]);
        pf.d[2 * t + 1] = pack2<DT>(x[t][2], x[t][3]);
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
  __syncthreads();
  for (int i = threadIdx.x * 4; i < rows * HD; i += 1024) {
    const int r = i / HD, d = i % HD;
    float top = sh_m[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, sh_m[w][r]);
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = exp2f(sh_m[w][r] - base);
      sum += sh_l[w][r] * a;
      acc += *(const f32x4*)(sh_o + (w * rows + r) * HD + d) * a;
    }
    const int64_t at = s * A.heads + h0 + r;
    if (whole) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      acc *= inv;
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
}

// The parts of a split context joined, one workgroup a (token, head): HD / 4
// lanes take the features, the lane groups every (1024 / HD)-th part.
template <int DT, int HD>
__global__ __launch_bounds__(256) void decode_join_kernel(PagedCache C, AttnArgs A) {
  constexpr int LN = HD / 4, NG = 256 / LN;
  __shared__ f32x4 sh_o[NG][LN];
  __shared__ float sh_l[NG];
  const int64_t s = blockIdx.y, at = s * A.heads + blockIdx.x;
  const int p = min(A.lengths[s], C.cols << C.log2_page) - 1;
  const TileRange range = tile_range<Shape<DT, HD>::T>(p, p, A.window, A.sinks);
  const int per = part_tiles(A, range.count);
  if (per >= range.count) return;  // the one part wrote the output
  const int parts = (range.count + per - 1) / per;
  const int d = threadIdx.x % LN, grp = threadIdx.x / LN;
  const float* ml = A.part_ml + 2 * at * A.n_split;
  const float* po = A.part_o + at * A.n_split * HD + 4 * d;
  float top = -INFINITY;
  for (int i = threadIdx.x & 63; i < parts; i += 64) top = fmaxf(top, ml[2 * i]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  for (int i = grp; i < parts; i += NG) {
    const float a = exp2f(ml[2 * i] - base);
    sum += ml[2 * i + 1] * a;
    acc += *(const f32x4*)(po + (int64_t)i * HD) * a;
  }
  sh_o[grp][d] = acc;
  if (d == 0) sh_l[grp] = sum;
  __syncthreads();
  if (grp) return;
  acc = sh_o[0][d];
  sum = sh_l[0];
#pragma unroll
  for (int i = 1; i < NG; ++i) {
    acc += sh_o[i][d];
    sum += sh_l[i];
  }
  acc *= sum == 0.f ? 0.f : 1.f / sum;
  if constexpr (DT == DT_F32)
    *(f32x4*)(A.out + (at * HD + 4 * d) * 4) = acc;
  else
    *(uint2*)(A.out + (at * HD + 4 * d) * 2) =
        uint2{pack2<DT>(acc[0], acc[1]), pack2<DT>(acc[2], acc[3])};
}

template <int DT, int HD>
void launch(const PagedCache& C, const AttnArgs& A, hipStream_t st) {
  const int G = A.heads / C.kv_heads;
  const int n_hb = (G + kHeadRows - 1) / kHeadRows;
  const size_t lds = 4 * sizeof(float) * HD * std::min(G, kHeadRows);
  const dim3 grid((unsigned)A.n_split, (unsigned)(C.kv_heads * n_hb), (unsigned)A.tokens);
  hipLaunchKernelGGL((decode_kernel<DT, HD>), grid, dim3(256), lds, st, C, A);
  if (A.n_split > 1)
    hipLaunchKernelGGL((decode_join_kernel<DT, HD>), dim3((unsigned)A.heads, (unsigned)A.tokens),
                       dim3(256), 0, st, C, A);
}

template <int DT>
void launch_dt(const PagedCache& C, const AttnArgs& A, hipStream_t st) {
  if (C.head_dim == 64) launch<DT, 64>(C, A, st);
  else if (C.head_dim == 128) launch<DT, 128>(C, A, st);
  else launch<DT, 256>(C, A, st);
}

}  // namespace

// Parts of about 1/2048 of the longest possible work, of 4 tiles (one a wave)
// at least. Fills n_split and per; returns the parts' bytes.
int64_t paged_decode_plan(const PagedCache& C, AttnArgs* A, int dtype, int64_t max_length) {
  const int T = dtype == SSL_F32 ? 16 : 32;
  const int G = A->heads / C.kv_heads;
  const int64_t blocks = A->tokens * C.kv_heads * ((G + kHeadRows - 1) / kHeadRows);
  int64_t reach = max_length;
  if (A->window)
    reach = std::min<int64_t>(reach, (int64_t)A->window + std::min(A->sinks, 0x3fffffff) + 2 * T);
  const int64_t tiles = std::max<int64_t>(1, (reach + T - 1) / T);
  int64_t per = std::max<int64_t>(4, (tiles * blocks + 2047) / 2048);
  per = (per + 3) / 4 * 4;
  A->per = (int)std::min<int64_t>(per, 0x3fffffff);
  A->n_split = (int)std::min<int64_t>((tiles + per - 1) / per, 65535);
  if (A->n_split <= 1) return 0;
  return A->tokens * A->heads * (int64_t)A->n_split * (C.head_dim + 2) * 4;
}

int paged_decode_launch(const PagedCache& C, const AttnArgs& A, int dtype, hipStream_t st) {
  if (dtype == SSL_F32) launch_dt<DT_F32>(C, A, st);
  else if (dtype == SSL_BF16) launch_dt<DT_BF16>(C, A, st);
  else launch_dt<DT_F16>(C, A, st);
  return check_hip(hipGetLastError(), "paged decode attention launch");
}

}  // namespace ssl
