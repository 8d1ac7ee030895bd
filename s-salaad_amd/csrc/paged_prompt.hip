// Attention of chunks of tokens over their sequences' pages: causal, with an
// optional window and first tokens that stay visible.
//
// 4·head_dim operations a (token, visible position, head): the matrix cores
// bound it. A row is one query head of one token; the rows of a key/value head
// are packed token by token (row r: token r / G, head r % G of the group), so
// short chunks of grouped heads fill the tiles and share what is loaded. A
// wave holds 32 rows, four waves (a team) 128; the teams of a workgroup take
// alternate tiles of KT positions and are joined through LDS.
//
//   Sᵀ = K·Qᵀ    32 keys × 32 rows a matrix instruction; a lane holds 16 keys of
//                one row, so its softmax needs one exchange between lane halves
//                and the running maximum and sum are scalars of a lane.
//   Oᵀ = Vᵀ·Pᵀ   P as the accumulators leave it (a contraction may take the keys
//                in any order both operands share); V is transposed on its way
//                out of LDS (ds_read_tr16), fp32 values are read as they are.
//
// What bounds it: 4096 tokens of one sequence, 16 heads of 128, bf16, hold a compute
// unit for 162000 cycles, 80 to 100 µs as the clock allows (2.1 to 1.7 GHz under it):
// 690 to 850 TFLOP/s (a large library product: 1157). 33 rounds of two tiles take 3870
// cycles each, in which a SIMD's two waves hold the matrix unit for 2048 and the vector
// unit for about as long, and the LDS works for a quarter; leaving out the loads, the
// exponentials, the sums or a product's three quarters saves 9 µs, 5, 3 or 13 each. The
// two waves pass the same barrier and want the same unit at a time, so a round is
// nearly the sum of both. (The teams half a round apart, by a second barrier: 3 µs
// more.) Beside its rounds a workgroup takes 17000 cycles: 4300 to its first loads, 5800
// for its first tile and q to arrive, 5200 to join its teams and store.
//
// 16-bit products take the weights rounded to the type; a row's sum is of the same
// rounded weights, two a dot product, so that their errors cancel where few weights
// carry a row: 4096 tokens are 2.04e-3 (rms) from 64 bits, at most 2.4e-3 of the
// largest, where one rounding of the result makes 1.65e-3 and 2.2e-3; with a sum of
// unrounded weights 2.14e-3 and 4.0e-3 in the same time. (Weights in two numbers, as
// few rows have them: 1.65e-3, and 117 µs for 93, launch after launch.)
//
// K and V go from memory into LDS directly, a tile ahead of its use, two
// buffers a team, one barrier a tile. LDS rows are permuted in 16-byte chunks by
// the row, so that fragment reads spread over the banks; the permutation is made
// by the address each lane loads. What lies past the last visible position or on
// no page is filled with zeros by the loads' bounds.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <utility>

#include "paged_join.h"

namespace ssl {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int DT, int HD>
struct Tile {
  static constexpr int EB = Elem<DT>::bytes;
  static constexpr bool F32 = DT == DT_F32;
  static constexpr int TEAMS = HD == 256 ? 1 : 2;
  static constexpr int KT = F32 ? 32 : 64;      // positions a tile
  static constexpr int ROWS = 128;              // rows a workgroup
  static constexpr int RB = HD * EB;            // bytes of an LDS row
  static constexpr int CPR = RB / 16;           // 16-byte chunks of a row
  static constexpr int RI = 1024 / RB;          // rows one load instruction fills
  static constexpr int IPG = 16 / RI;           // instructions a group of 16 rows
  static constexpr int NQ = IPG / 4 > 0 ? IPG / 4 : 1;
  static constexpr int BUF = KT * RB;           // one of K, V
  static constexpr int LDS = TEAMS * 4 * BUF;
  static constexpr int THREADS = TEAMS * 256;
  static constexpr int KS = KT / 32;
  static constexpr int QS = HD / (F32 ? 8 : 16);  // contraction steps of Sᵀ
  static constexpr int OT = HD / 32;              // output tiles
  // the chunk permutation of row r (of a group of 16)
  __device__ static int swz_k(int r) { return CPR == 8 ? (r >> 1) & 7 : r & 15; }
  // (V: pairs of chunks; a transposing read takes 4 rows × 2 pairs at a time)
  __device__ static int swz_v(int r) {
    return F32 ? 0 : ((CPR == 8 ? r & 2 : (r & 3) << 1) | (r >> 2 & 1)) << 1;
  }
};

// 16 bytes a lane from memory into LDS (lane l: lds + OFF + 16·l), zeros past the
// resource's size. In assembly, so that the compiler adds no waits of its own
// for it: wait_loads and the barrier below order it. (s_nop: the load takes m0 one wait
// state after a scalar write and its resource five after a vector one, which the
// compiler cannot see to here; with one state or four the times are the same.)
template <int OFF>
__device__ __forceinline__ void dma16(const u32x4& r, uint32_t voff, uint32_t lds) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(r), "n"(OFF)
               : "m0", "scc");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// 4 elements of column l % 16 of the 4 × 16 block a group of 16 lanes addresses
// (lane l: row l / 4, 4 elements from 4·(l % 4))
__device__ __forceinline__ uint2 read_tr(uint32_t lds) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)(uintptr_t)lds));
}
__device__ __forceinline__ uint4 read16(uint32_t lds) {
  return __builtin_bit_cast(uint4, *(__attribute__((address_space(3))) u32x4*)(uintptr_t)lds);
}
__device__ __forceinline__ uint2 read8(uint32_t lds) {
  return __builtin_bit_cast(uint2, *(__attribute__((address_space(3))) u32x2*)(uintptr_t)lds);
}

// to and the two 16-bit elements of a pair
template <int DT>
__device__ __forceinline__ float sum2(uint32_t pair, float to) {
  if constexpr (DT == DT_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair),
                                           bf16x2{(__bf16)1.f, (__bf16)1.f}, to, false);
  } else {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair),
                                  f16x2{(_Float16)1.f, (_Float16)1.f}, to, false);
  }
}
template <int DT>
__device__ __forceinline__ void mma(f32x16& acc, const uint4& a, const uint4& b) {
  if constexpr (DT == DT_BF16)
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                  __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  else
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                 __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
}
__device__ __forceinline__ void mma_f32(f32x16& acc, float a, float b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, acc, 0, 0, 0);
}

// Where paths meet, keeps accumulators in the registers the matrix instructions
// use. (Else each path leaves its elements in registers of its own, which are
// copied, 16 a vector, and held twice.)
template <int N>
__device__ __forceinline__ void whole_registers(f32x16 (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm("" : "+v"(v[i]));
}

template <typename F, int... I>
__device__ __forceinline__ void unroll_over(F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unroll(F f) {
  unroll_over(f, std::make_integer_sequence<int, N>{});
}

// The u-th row tile of all chunks, later tiles of their chunks (the longest
// contexts) first: its sequence and tile, or a sequence of -1 past the last. Each
// wave finds it by itself, a lane a sequence: N(t), the tiles numbered t or above,
// by sums over the lanes, the tile number by bisection, the sequence by counting.
template <int ROWS>
__device__ __forceinline__ Chunk find_tile(const PagedCache& C, const AttnArgs& A, int G, int u,
                                           int lane, int* seq, int* tile) {
  struct Span {
    int a, b;
  };
  const auto span_of = [&](int s) {
    const int n = (int)A.tokens;
    const int a = s == 0 || s >= C.seqs ? 0 : min(max(A.cu[s], 0), n);
    return Span{a, s >= C.seqs ? 0 : min(max(A.cu[s + 1], a), n)};
  };
  const auto tiles_of = [&](Span x) { return ((x.b - x.a) * G + ROWS - 1) / ROWS; };
  const Span mine = span_of(lane);  // of the first 64 sequences, kept
  const int length = A.lengths[min(lane, C.seqs - 1)];
  const int first = tiles_of(mine);
  const auto from = [&](int t) {  // N(t)
    int n = max(first - t, 0);
    for (int s = 64 + lane; s < C.seqs; s += 64) n += max(tiles_of(span_of(s)) - t, 0);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o);
    return __builtin_amdgcn_readfirstlane(n);
  };
  int s = -1;
  if (C.seqs == 1) {
    const int n = __builtin_amdgcn_readfirstlane(first);
    *tile = n - 1 - u;
    if (u < n) s = 0;
  } else if (from(0) > u) {
    int lo = 0, hi = (int)((A.tokens * G + ROWS - 1) / ROWS);  // N(lo) > u >= N(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (from(mid) > u) lo = mid;
      else hi = mid;
    }
    *tile = lo;
    int left = u - from(hi);  // chunks with a tile lo before it
    for (int s0 = 0; s0 < C.seqs && s < 0; s0 += 64) {
      uint64_t has = __ballot((s0 ? tiles_of(span_of(s0 + lane)) : first) > lo);
      const int count = __popcll(has);
      if (left < count) {
        for (; left > 0; --left) has &= has - 1;
        s = s0 + __builtin_ctzll(has);
      }
      left -= count;
    }
  }
  *seq = s;
  if (s >= 64) return Chunk(C, A, s, G);
  s = max(s, 0);
  return Chunk(C, __builtin_amdgcn_readlane(mine.a, s), __builtin_amdgcn_readlane(mine.b, s),
               __builtin_amdgcn_readlane(length, s), G);
}

template <int DT, int HD>
__global__ __launch_bounds__((Tile<DT, HD>::THREADS)) void prompt_kernel(PagedCache C, AttnArgs A,
                                                                          int64_t n_tiles) {
  using T = Tile<DT, HD>;
  extern __shared__ char lds[];
  const int G = A.heads / C.kv_heads;
  // key/value heads fastest (one head's K and V stay in one die's cache where
  // their number is a multiple of 8); after the row tiles a workgroup a head for
  // the tokens past the last chunk. (Workgroups that end at once come last:
  // between the others they would leave shader engines idle, to which workgroups
  // go in turn.)
  uint32_t id = blockIdx.x;
  const int kh = id % C.kv_heads;
  id /= C.kv_heads;
  const int split = id % A.n_split;
  id /= A.n_split;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int team = wave >> 2, w = wave & 3;
  const int col = lane & 31, h = lane >> 5;

  if (id >= n_tiles) {
    if (split == 0) zero_tail(C, A, kh, T::CPR, tid, T::THREADS);
    return;
  }
  int s, tile;
  const Chunk chunk = find_tile<T::ROWS>(C, A, G, (int)id, lane, &s, &tile);
  if (s < 0) return;
  const int32_t* table = C.table + (int64_t)s * C.table_stride;
  const uint32_t slot_bytes = (uint32_t)(C.slot_stride * T::EB);
  const uint64_t page_bytes = (uint64_t)C.page_stride * T::EB;
  const uint64_t k_base = (uint64_t)(uintptr_t)C.k + kh * C.head_stride * T::EB;
  const uint64_t v_base = (uint64_t)(uintptr_t)C.v + kh * C.head_stride * T::EB;
  constexpr float kBias = DT == DT_F16 ? 4.f : 0.f;  // fp16 weights are kept 16-fold
  constexpr bool kRoundAll = HD == 256;              // scores, before their weights

  const int row_a = tile * T::ROWS, row_b = min(row_a + T::ROWS, chunk.rows) - 1;
  const int p_min = chunk.p0 + row_a / G, p_max = chunk.p0 + row_b / G;
  const TileRange range = tile_range<T::KT>(max(p_min, 0), p_max, A.window, A.sinks);
  const int per = part_tiles(A, range.count);
  const bool whole = per >= range.count;
  const int lo = split * per, hi = min(lo + per, range.count);
  if (lo >= hi && split > 0) return;
  const int limit = p_max + 1;
  const int w_first = A.window && p_min + 1 > A.window ? p_min + 1 - A.window : 0;

  // this wave's rows
  const int r_a = row_a + w * 32;
  const bool any = r_a <= row_b;
  const int r = min(r_a + col, row_b);
  const int64_t token = chunk.t0 + r / G;
  const int head = kh * G + r % G;
  const int p = chunk.p0 + r / G;
  const int first = A.window && p + 1 > A.window ? p + 1 - A.window : 0;
  const int wp_min = chunk.p0 + r_a / G, wp_max = chunk.p0 + min(r_a + 31, row_b) / G;
  const int wfirst_max = A.window && wp_max + 1 > A.window ? wp_max + 1 - A.window : 0;

  uint4 qf[T::QS];
  f32x16 o[T::OT];
#pragma unroll
  for (int i = 0; i < T::OT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  const uint32_t lds0 = lds_addr(lds) + team * 4 * T::BUF;
  // load lanes: LDS chunk lane % CPR of row lane / CPR of an instruction
  uint32_t k_off[T::NQ], v_off[T::NQ];
  int l_row[T::NQ];
#pragma unroll
  for (int q = 0; q < T::NQ; ++q) {
    const int r16 = (T::IPG >= 4 ? (q * 4 + w) * T::RI : (w & 1) * T::RI) + lane / T::CPR;
    l_row[q] = r16;
    k_off[q] = r16 * slot_bytes + ((lane % T::CPR) ^ T::swz_k(r16)) * 16;
    v_off[q] = r16 * slot_bytes + ((lane % T::CPR) ^ T::swz_v(r16)) * 16;
  }
  // page of group lane % (KT / 16) of tile i
  auto pages_of = [&](int i) {
    const int key = range.tile(min(i, hi - 1)) * T::KT + 16 * (lane % (T::KT / 16));
    return table[min(key >> C.log2_page, C.cols - 1)];
  };
  // The next tile's loads. Each lane settles one group of 16 positions (group
  // lane % (KT / 16)): its place in the pools and the bytes of it that are
  // loaded; load<I> reads them from that lane and issues the wave's I-th loads of
  // K and V. A tile that does not exist loads zeros.
  constexpr int KG = T::KT / 16;
  constexpr int LOADS = (T::IPG >= 4 ? KG : KG / 2) * T::NQ;
  uint64_t off_l = 0;
  uint32_t size_l = 0, next_lds = 0, hide_span = 0;
  int hide_from = 0;
  auto next_tile = [&](int i, int buf, int32_t page) {
    const int key0 = range.tile(i) * T::KT;
    const int key_l = key0 + 16 * (lane % KG);
    const bool has = C.has(page) && i < hi;
    off_l = (uint64_t)(uint32_t)(has ? page : 0) * page_bytes +
            (uint32_t)(key_l & (C.page - 1)) * slot_bytes;
    size_l = has ? min(max(limit - key_l, 0), 16) * slot_bytes : 0u;
    next_lds = lds0 + 2 * buf * T::BUF + w * 1024;
    // positions from sinks to the window's first: zeros as well
    hide_from = key0 - A.sinks;
    hide_span = key0 < w_first ? max(w_first - A.sinks, 0) : 0;
  };
  auto load = [&](auto at) {
    constexpr int n = decltype(at)::value / T::NQ, q = decltype(at)::value % T::NQ;
    const int grp = T::IPG >= 4 ? n : 2 * n + (w >> 1);
    const uint64_t off =
        ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(off_l >> 32), grp) << 32) |
        (uint32_t)__builtin_amdgcn_readlane((int)off_l, grp);
    const uint64_t ka = k_base + off, va = v_base + off;
    u32x4 rk, rv;
    rk[0] = (uint32_t)ka;
    rk[1] = (uint32_t)(ka >> 32);
    rv[0] = (uint32_t)va;
    rv[1] = (uint32_t)(va >> 32);
    rk[2] = rv[2] = __builtin_amdgcn_readlane((int)size_l, grp);
    rk[3] = rv[3] = 0x00020000u;
    const uint32_t hide =
        (uint32_t)(hide_from + 16 * grp + l_row[q]) < hide_span ? 0x80000000u : 0u;
    // the instruction fills 1 KiB at n · max(IPG, 4) + 4 q + w
    constexpr int to = (n * (T::IPG >= 4 ? T::IPG : 4) + 4 * q) * 1024;
    dma16<to>(rk, k_off[q] | hide, next_lds);
    dma16<to + T::BUF>(rv, v_off[q] | hide, next_lds);
  };

  // Fragment addresses in the first buffer: step k of a K row and output tile d
  // of V differ by an exclusive or below 256 bytes (the permutation's reach) and
  // by a plain offset above; the buffers' parity is one more bit to flip.
  constexpr int KX = std::min(T::QS, T::RB >= 256 ? 8 : 4);
  constexpr int VX = T::F32 ? 1 : std::min(T::OT, 4);
  uint32_t kx[KX], vx[VX];
#pragma unroll
  for (int k = 0; k < KX; ++k)
    kx[k] = lds0 + col * T::RB + (((h ^ T::swz_k(col & 15)) * 16) ^ (k * 32));
  if constexpr (T::F32) {
    vx[0] = lds0 + T::BUF + 4 * h * T::RB + col * (HD == 64 ? 8 : 16);
  } else {
    const int vr = 4 * h + ((lane & 15) >> 2);
#pragma unroll
    for (int d = 0; d < VX; ++d)
      vx[d] = lds0 + T::BUF + vr * T::RB + (lane & 3) * 8 +
              (((((lane >> 4) & 1) * 2) ^ T::swz_v(vr) ^ (4 * d)) * 16);
  }
  auto read_k = [&](int f) {  // fragment f = t · QS + k
    const int t = f / T::QS, k = f % T::QS;
    return read16(kx[k % KX] + (k / KX) * KX * 32 + t * 32 * T::RB);
  };
  auto read_v = [&](int f) {  // fragment f = j · OT + d
    const int j = f / T::OT, d = f % T::OT;
    const uint32_t at = vx[d % VX] + (d / VX) * VX * 64 + 16 * j * T::RB;
    const uint2 a = read_tr(at), b = read_tr(at + 8 * T::RB);
    return uint4{a.x, a.y, b.x, b.y};
  };
  // One tile of the wave's rows. Fragments are read kAhead before their product
  // and the order is pinned: left alone the compiler reads each right before
  // its product and waits. Each step of the second product computes the weights
  // of the next.
  constexpr int kAhead = 4;
  auto tile_step = [&](int key0, uint32_t bad, bool all) {
    constexpr int KF = T::KS * T::QS;
    f32x16 x[T::KS];
#pragma unroll
    for (int t = 0; t < T::KS; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[t][e] = 0.f;
    {
      uint4 f[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) f[i] = read_k(i);
      __builtin_amdgcn_sched_barrier(0);
      unroll<KF>([&](auto at) {
        constexpr int i = decltype(at)::value;
        const uint4 kf = f[i % kAhead], q = qf[i % T::QS];
        f32x16& acc = x[i / T::QS];
        if constexpr (T::F32) {
          mma_f32(acc, __uint_as_float(kf.x), __uint_as_float(q.x));
          mma_f32(acc, __uint_as_float(kf.y), __uint_as_float(q.y));
          mma_f32(acc, __uint_as_float(kf.z), __uint_as_float(q.z));
          mma_f32(acc, __uint_as_float(kf.w), __uint_as_float(q.w));
        } else {
          mma<DT>(acc, kf, q);
        }
        if constexpr (i + kAhead < KF) f[i % kAhead] = read_k(i + kAhead);
        if constexpr (i % (KF / LOADS) == 1)
          load(std::integral_constant<int, i / (KF / LOADS)>{});
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    constexpr int VF = 2 * T::KS * T::OT;
    uint4 vf[T::F32 ? 1 : kAhead];
    if constexpr (!T::F32) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) vf[i] = read_v(i);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!all) {
#pragma unroll
      for (int t = 0; t < T::KS; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = key0 + 32 * t + 8 * (e >> 2) + 4 * h + (e & 3);
          const bool see = key <= p && (key >= first || key < A.sinks) &&
                           !((bad >> (2 * t + (e >> 3))) & 1);
          x[t][e] = see ? x[t][e] : -INFINITY;
        }
    }
    whole_registers(x);
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < T::KS; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, x[t][e]);
    {  // with the row's other lane
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx),
                                                         false, false);
      mx = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * A.scale_log2;
    }
    // o and l keep an older maximum while it is at most 2^8 too small: the
    // weights stay in range and most tiles need no scaling
    if (__any(mx - m > 8.f)) {
      const float top = fmaxf(m, mx);
      const float a = exp2f(m - (top == -INFINITY ? 0.f : top));
      l *= a;
#pragma unroll
      for (int d = 0; d < T::OT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= a;
      m = top;
    }
    // Weights: a fused product minus the maximum, or of scores rounded first. The
    // 256-wide heads, whose registers are all taken, always round them (2000 tokens,
    // 8 heads: 55 µs, with a path for far scores 56), the others only far from
    // zero (4096 tokens, 16 heads of 128: no difference, always: 1.5 µs of 93).
    const float top = m == -INFINITY ? 0.f : m;
    float scale = A.scale_log2, base = top - kBias;
    if constexpr (!kRoundAll) {
      const bool far = fabsf(top) >= kFarScore;
      if (__any(far)) {
#pragma unroll
        for (int t = 0; t < T::KS; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            x[t][e] = far ? rounded(x[t][e] * A.scale_log2) - top : x[t][e];
        scale = far ? 1.f : scale;
        base = far ? -kBias : base;
      }
      whole_registers(x);
    }
    auto weight = [&](int i) {
      const float z = x[i >> 4][i & 15];
      const float y = __builtin_amdgcn_exp2f(kRoundAll ? rounded(z * scale) - top + kBias
                                                       : fmaf(z, scale, -base));
      x[i >> 4][i & 15] = y;
      if constexpr (T::F32) l += y;
    };
    if constexpr (T::F32) {
#pragma unroll
      for (int i = 0; i < 16 * T::KS; ++i) weight(i);
#pragma unroll
      for (int t = 0; t < T::KS; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t at = vx[0] + (32 * t + 8 * (e >> 2) + (e & 3)) * T::RB;
          if constexpr (HD == 64) {
            const uint2 v = read8(at);
            mma_f32(o[0], __uint_as_float(v.x), x[t][e]);
            mma_f32(o[1], __uint_as_float(v.y), x[t][e]);
          } else {
#pragma unroll
            for (int d = 0; d < T::OT; d += 4) {
              const uint4 v = read16(at + d * 128);
              mma_f32(o[d], __uint_as_float(v.x), x[t][e]);
              mma_f32(o[d + 1], __uint_as_float(v.y), x[t][e]);
              mma_f32(o[d + 2], __uint_as_float(v.z), x[t][e]);
              mma_f32(o[d + 3], __uint_as_float(v.w), x[t][e]);
            }
          }
        }
    } else {
      auto packed = [&](int j) {
        const f32x16& y = x[j >> 1];
        const int e = 8 * (j & 1);
        const uint4 r{pack2<DT>(y[e], y[e + 1]), pack2<DT>(y[e + 2], y[e + 3]),
                      pack2<DT>(y[e + 4], y[e + 5]), pack2<DT>(y[e + 6], y[e + 7])};
        l = sum2<DT>(r.x, l);
        l = sum2<DT>(r.y, l);
        l = sum2<DT>(r.z, l);
        l = sum2<DT>(r.w, l);
        return r;
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) weight(i);
      uint4 pf = packed(0);
#pragma unroll
      for (int i = 0; i < VF; ++i) {
        const int j = i / T::OT, d = i % T::OT;
        mma<DT>(o[d], vf[i % kAhead], pf);
        if (i + kAhead < VF) vf[i % kAhead] = read_v(i + kAhead);
        if (j + 1 < 2 * T::KS) {
#pragma unroll
          for (int k = 8 * d / T::OT; k < 8 * (d + 1) / T::OT; ++k) weight(8 * (j + 1) + k);
          if (d == T::OT - 1) pf = packed(j + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  const int rounds = (hi - lo + T::TEAMS - 1) / T::TEAMS;
  int32_t pgv = 0;
  uint32_t bad_next = 0;  // groups of 16 of the tile that lie on no page
  auto missing = [&](int32_t pg) {
    return (uint32_t)__ballot(!C.has(pg)) & ((1u << (T::KT / 16)) - 1);
  };
  if (rounds > 0) {
    pgv = pages_of(lo + team);
    bad_next = missing(pgv);
    next_tile(lo + team, 0, pgv);
    unroll<LOADS>(load);
    pgv = pages_of(lo + team + T::TEAMS);
  }
#pragma unroll
  for (int i = 0; i < T::QS; ++i) {  // after the first tile's loads, to arrive with them
    qf[i] = *(const uint4*)(A.q + (token * A.q_token + (int64_t)head * A.q_head) * T::EB +
                            (2 * i + h) * 16);
    const uint32_t flip = A.flip & (T::F32 ? 0x80000000u : 0x80008000u);
    qf[i] = uint4{(qf[i].x & A.keep) ^ flip, (qf[i].y & A.keep) ^ flip,
                  (qf[i].z & A.keep) ^ flip, (qf[i].w & A.keep) ^ flip};
  }
  if (!any) {  // a wave without rows only loads
    for (int n = 0; n < rounds; ++n) {
      const int i = lo + n * T::TEAMS + team;
      wait_loads();
      barrier();
      next_tile(i + T::TEAMS, (n + 1) & 1, pgv);
      pgv = pages_of(i + 2 * T::TEAMS);
      unroll<LOADS>(load);
    }
  } else {
    for (int n = 0; n < rounds; ++n) {
      const int i = lo + n * T::TEAMS + team;
      wait_loads();
      barrier();
      // a tile past the end, or seen by no row, runs masked: its workgroup waits
      // for the others' anyway, and a path around it costs copies of o
      const uint32_t bad = i < hi ? bad_next : ~0u;
      bad_next = missing(pgv);
      next_tile(i + T::TEAMS, (n + 1) & 1, pgv);
      pgv = pages_of(i + 2 * T::TEAMS);
      const int key0 = range.tile(i) * T::KT;
      const bool all = key0 + T::KT - 1 <= wp_min && !bad &&
                       (key0 >= wfirst_max || key0 + T::KT <= A.sinks);
      tile_step(key0, bad, all);
#pragma unroll
      for (int k = 0; k < KX; ++k) kx[k] ^= 2 * T::BUF;  // the other buffers
#pragma unroll
      for (int k = 0; k < VX; ++k) vx[k] ^= 2 * T::BUF;
    }
  }
  wait_loads();
  l += __shfl_xor(l, 32);

  // The teams' parts are joined, each team half of the output tiles: it leaves
  // the other's half in LDS and takes its own from there.
  constexpr int HALF = T::OT / T::TEAMS;
  if constexpr (T::TEAMS == 2) {
    barrier();
    f32x4* part = (f32x4*)lds + (w * HALF * 4) * 64 + lane;  // [team][wave][tile][4][lane]
    float* ml = (float*)(lds + 2 * 4 * HALF * 4 * 64 * 16) + w * 128 + lane;
    constexpr int STEP = 4 * HALF * 4 * 64;
#pragma unroll
    for (int d = 0; d < HALF; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = team ? o[d][4 * k + e] : o[HALF + d][4 * k + e];
        part[team * STEP + (d * 4 + k) * 64] = y;
      }
    ml[team * 512] = m;
    ml[team * 512 + 64] = l;
    barrier();
    const float m2 = ml[(team ^ 1) * 512], l2 = ml[(team ^ 1) * 512 + 64];
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    const float a = exp2f(m - base), b = exp2f(m2 - base);
    // in the order of the teams, so that both halves have one l
    l = team ? l2 * b + l * a : l * a + l2 * b;
    m = top;
#pragma unroll
    for (int d = 0; d < HALF; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 y = part[(team ^ 1) * STEP + (d * 4 + k) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[d][4 * k + e] = (team ? o[HALF + d][4 * k + e] : o[d][4 * k + e]) * a + y[e] * b;
      }
  }
  const int64_t at = token * A.heads + head;
  const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
  if (r_a + col <= row_b) {
    if (!whole && h == 0 && team == 0) {
      float* ml = A.part_ml + 2 * (at * A.n_split + split);
      ml[0] = m;
      ml[1] = l;
    }
    // 4 adjacent features at a time, or one
    auto put1 = [&](int f, float y) {
      float* to = whole ? (float*)A.out + at * HD : A.part_o + (at * A.n_split + split) * HD;
      to[f] = y;
    };
    auto put = [&](int f, const f32x4 y) {
      if (!whole)
        *(f32x4*)(A.part_o + (at * A.n_split + split) * HD + f) = y;
      else if constexpr (T::F32)
        *(f32x4*)(A.out + (at * HD + f) * 4) = y;
      else
        *(uint2*)(A.out + (at * HD + f) * 2) = uint2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
    };
    if constexpr (!T::F32) {
      // 8 adjacent features a lane, its own 4 and the row's other lane's: the stores
      // of 128 rows 4 KB apart took 4800 cycles of 4 features each, 1.2 µs of 83 at
      // 4096 tokens
      if (whole) {
#pragma unroll
        for (int d = 0; d < HALF; ++d)
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              y[i] = pack2<DT>(o[d][4 * k + 2 * i] * inv, o[d][4 * k + 2 * i + 1] * inv);
            const auto a = __builtin_amdgcn_permlane32_swap(y[0], y[2], false, false);
            const auto b = __builtin_amdgcn_permlane32_swap(y[1], y[3], false, false);
            *(uint4*)(A.out + (at * HD + 32 * (team * HALF + d) + 8 * (k + h)) * 2) =
                uint4{a[0], b[0], a[1], b[1]};
          }
      } else {
#pragma unroll
        for (int d = 0; d < HALF; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            put(32 * (team * HALF + d) + 8 * k + 4 * h,
                f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]} * inv);
      }
    } else {
      // fp32: feature f of a lane's vector lies in output tile f, so a team holds
      // HALF adjacent ones
      constexpr int VE = std::min(T::OT, 4);
#pragma unroll
      for (int d = 0; d < HALF; d += 4)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int f = 32 * d + VE * (8 * (e >> 2) + 4 * h + (e & 3)) + team * HALF;
          if constexpr (HALF >= 4) {
            put(f, f32x4{o[d][e], o[d + 1][e], o[d + 2][e], o[d + 3][e]} * inv);
          } else {
#pragma unroll
            for (int i = 0; i < HALF; ++i) put1(f + i, o[i][e] * inv);
          }
        }
    }
  }

  float finite = 0.f;
#pragma unroll
  for (int d = 0; d < HALF; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) finite = fmaf(o[d][e], 0.f, finite);
  // (a row whose sum is NaN is NaN by its own scores)
  const uint64_t lanes = __ballot(r_a + col <= row_b && finite != 0.f && l == l);
  uint32_t anew = (uint32_t)(lanes | lanes >> 32);
  if (!anew) return;
  wait_loads();  // and the stores above
  for (; anew; anew &= anew - 1) {
    const int c = __builtin_ctz(anew), rc = r_a + c;
    const int64_t tc = chunk.t0 + rc / G;
    const int hc = kh * G + rc % G;
    const float lc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l), c));
    row_anew<DT, HD, T::KT>(
        C, A, s, kh, tc, hc, chunk.p0 + rc / G, range, lo, hi, lc,
        whole ? nullptr : A.part_o + ((tc * A.heads + hc) * A.n_split + split) * HD,
        [&](int f) {  // the team's own
          return T::TEAMS == 1 || (T::F32 ? f / HALF % 2 : f / (HD / 2)) == team;
        });
  }
}

template <int DT, int HD>
int launch(const PagedCache& C, const AttnArgs& A, hipStream_t st) {
  using T = Tile<DT, HD>;
  // row tiles at most: a partly filled one a sequence. (None without sequences, of
  // which a tile's workgroup reads lengths: only the tokens past the last chunk.)
  const int64_t n_tiles =
      C.seqs ? A.tokens * (A.heads / C.kv_heads) / T::ROWS + C.seqs : 0;
  const int64_t grid = (n_tiles + 1) * A.n_split * C.kv_heads;
  if (grid > 0x7fffffff)
    return fail(SSL_ERR_UNSUPPORTED, "paged_attention: a grid of %lld workgroups", (long long)grid);
  if (T::LDS > 64 * 1024) {
    static std::atomic<uint64_t> raised{0};
    if (int rc = allow_lds((const void*)prompt_kernel<DT, HD>, T::LDS, &raised)) return rc;
  }
  hipLaunchKernelGGL((prompt_kernel<DT, HD>), dim3((unsigned)grid), dim3(T::THREADS), T::LDS, st, C,
                     A, n_tiles);
  if (A.n_split > 1) launch_join<DT, HD, T::KT, T::ROWS>(C, A, st);
  return SSL_OK;
}

template <int DT>
int launch_dt(const PagedCache& C, const AttnArgs& A, hipStream_t st) {
  if (C.head_dim == 64) return launch<DT, 64>(C, A, st);
  if (C.head_dim == 128) return launch<DT, 128>(C, A, st);
  return launch<DT, 256>(C, A, st);
}

}  // namespace

// Splits contexts where that is faster by an estimate of the launch: a round (a tile
// a team) takes kRound µs with its share of what a workgroup does beside them, a
// compute unit takes one workgroup at a time (64-wide heads leave LDS for two, but
// their registers, 138 and 159, hold no more than 12 waves), and a join costs 4 µs and
// its parts' traffic at 3 TB/s. A device full of 64-wide heads waits a third of its
// last parts besides. (2 prompts of 1000 tokens, 16 heads of 128: whole 23 µs, in 2
// parts 38; 500 tokens, 8 fp32 heads of 128: whole 74 µs, in 4 parts 35, in 8 32; 4096
// tokens, 16 heads of 64: whole 64 µs, in 2 parts 112; 250 over 4000 positions, 16
// heads of 64 over 4: whole 46 µs, in 6 parts 21.) Fills n_split and per; returns the
// parts' bytes.
int64_t paged_prompt_plan(const PagedCache& C, AttnArgs* A, int dtype, int64_t max_tokens,
                          int64_t max_length) {
  // by head_dim 64, 128, 256
  static constexpr double kRound[2][3] = {{1.4, 2.2, 2.8}, {5.5, 7.6, 8.9}};
  const bool f32 = dtype == SSL_F32;
  const int KT = f32 ? 32 : 64, G = A->heads / C.kv_heads;
  const int teams = C.head_dim == 256 ? 1 : 2;
  const double slots = (double)device_cus(), tail = C.head_dim == 64 ? 1. / 3 : 0.;
  const double round = kRound[f32][C.head_dim == 64 ? 0 : C.head_dim == 128 ? 1 : 2];
  const int64_t per_seq = std::max<int64_t>(1, (max_tokens * G + 127) / 128);
  const int64_t tiles = std::min<int64_t>(C.seqs * per_seq, A->tokens * G / 128 + C.seqs);
  const int64_t blocks = std::max<int64_t>(1, tiles * C.kv_heads);
  int64_t reach = max_length;
  double mean = 1 - 0.5 * max_tokens / std::max<double>(1, max_length);  // of the rows' contexts
  if (A->window) {
    reach = std::min<int64_t>(reach, (int64_t)A->window + std::min(A->sinks, 0x3fffffff) +
                                         128 / G + 2 * KT);
    mean = 1;
  }
  const int64_t keys = std::max<int64_t>(1, (reach + KT - 1) / KT);
  const double part_us = A->tokens * A->heads * (double)C.head_dim * 8 / 3e6;
  double best = 0;
  for (int n = 1; n <= 64 && (n == 1 || n <= keys); n += n < 4 ? 1 : n / 2) {
    const int64_t per = (keys + n - 1) / n, parts = (keys + per - 1) / per;
    const double rounds = (double)((per + teams - 1) / teams);
    const double full = blocks * mean * keys / teams / slots;
    const double us = round * std::max(rounds, full + tail * rounds) + (parts > 1 ? 4 + parts * part_us : 0);
    if (n == 1 || us < best) {
      best = us;
      A->per = (int)std::min<int64_t>(per, 0x3fffffff);
      A->n_split = (int)parts;
    }
  }
  A->us = (float)(7 + best);
  if (A->n_split <= 1) return 0;
  return A->tokens * A->heads * (int64_t)A->n_split * (C.head_dim + 2) * 4;
}

int paged_prompt_launch(const PagedCache& C, const AttnArgs& A, int dtype, hipStream_t st) {
  int rc;
  if (dtype == SSL_F32) rc = launch_dt<DT_F32>(C, A, st);
  else if (dtype == SSL_BF16) rc = launch_dt<DT_BF16>(C, A, st);
  else rc = launch_dt<DT_F16>(C, A, st);
  return rc ? rc : check_hip(hipGetLastError(), "paged prompt attention launch");
}

}  // namespace ssl
