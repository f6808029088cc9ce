// bb_paged.hip — rotary positions, appending to a paged key/value cache, and attention of one new
// token per sequence over it (include/bebelm_moe.h states the operators). The reference has no
// counterpart: values are computed in f32 from the formulas and rounded once where they are stored.
#include "bb_device.h"
#include <algorithm>
#include <type_traits>
#include "bb_internal.h"
#include "bb_paged_plan.h"

namespace bb {

namespace {

template <int DT>
struct ElemOf;
template <>
struct ElemOf<BB_F32> {
  typedef float T;
};
template <>
struct ElemOf<BB_F16> {
  typedef _Float16 T;
};
template <>
struct ElemOf<BB_BF16> {
  typedef __bf16 T;
};

// N consecutive elements at any element's alignment as f32, and back, rounded to nearest (16-byte accesses).
template <class T, int N>
struct RunOf {
  static constexpr int M = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
  typedef T V __attribute__((ext_vector_type(M), aligned(sizeof(T))));
};
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = (float)p[0];
  } else {
    constexpr int M = RunOf<T, N>::M;
#pragma unroll
    for (int i = 0; i < N; i += M) {
      const auto v = *reinterpret_cast<const typename RunOf<T, N>::V*>(p + i);
#pragma unroll
      for (int j = 0; j < M; ++j) x[i + j] = (float)v[j];
    }
  }
}
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  if constexpr (N == 1) {
    p[0] = (T)x[0];
  } else {
    constexpr int M = RunOf<T, N>::M;
#pragma unroll
    for (int i = 0; i < N; i += M) {
      typename RunOf<T, N>::V v;
#pragma unroll
      for (int j = 0; j < M; ++j) v[j] = (T)x[i + j];
      *reinterpret_cast<typename RunOf<T, N>::V*>(p + i) = v;
    }
  }
}

// i / page_slots for 0 <= i < 2^31.
__device__ __forceinline__ int page_of(const PagedView& kv, int i) {
  return slot_quotient(i, kv.page_mul, kv.page_shift);
}

// ---- rotary positions, and the rows of an append ------------------------------------------------

// (cos, sin) of pos·f, f given as turns per position: the angle is reduced in f64 to a quarter turn's
// fraction in ±1/2 (exact but for the product's rounding: 2^-53 of the turns), so that its rounding to
// f32 costs at most 2^-26·pi/2 = 2^-25.3 of the values, whatever the position.
__device__ __forceinline__ float2 cos_sin_turns(int pos, double turns) {
  const double q4 = 4.0 * ((double)pos * turns);
  const double n = rint(q4);
  float s, c;
  sincospif(0.5f * (float)(q4 - n), &s, &c);
  const double w = n - 4.0 * floor(0.25 * n);  // n mod 4
  const int k = (int)w;
  const float cc = (k & 1) ? -s : c, ss = (k & 1) ? c : s;
  return (k & 2) ? make_float2(-cc, -ss) : make_float2(cc, ss);
}

constexpr int RR_THREADS = 256;

struct RowPlace {
  int64_t base;  // where its keys and values start in the pool, -1: nowhere
  int pos;
  int live;
};

// The place and position of token t. Called by a whole wave; every lane gets the answer.
__device__ __forceinline__ RowPlace row_place(const RopeRows& r, const PagedView& kv, const PagedSeqs& sq, size_t t) {
  RowPlace w{-1, 0, 0};
  if (t >= r.T) return w;
  if (!sq.lens) {
    w.pos = r.pos[t];
    w.live = 1;
    return w;
  }
  int s = (int)t;
  int64_t index;
  if (r.seq_start) {
    // the sequence is the number of sequences that end at or before t (64 at a time)
    const int lane = threadIdx.x & 63;
    s = 0;
    for (int b = 0; b < sq.n_seqs; b += 64) {
      const int i = b + lane;
      const bool before = i < sq.n_seqs && r.seq_start[i + 1] <= (int64_t)t;
      s += __popcll(__ballot(before));
    }
    if (s >= sq.n_seqs) return w;
    index = (int64_t)sq.lens[s] - r.seq_start[s + 1] + (int64_t)t;
  } else {
    index = (int64_t)sq.lens[s] - 1;
  }
  if (index < 0 || index >= (int64_t)sq.max_pages * kv.page_size) return w;
  const int ix = (int)index, page = page_of(kv, ix);
  w.live = 1;
  w.pos = r.pos ? r.pos[t] : ix;
  if (r.n_kv) {
    const int pg = sq.table[(size_t)s * sq.table_stride + page];
    if (pg >= 0 && pg < kv.n_pages)
      w.base = (int64_t)((size_t)pg * kv.page_stride + (size_t)(ix - page * kv.page_size) * kv.pos_stride);
  }
  return w;
}

// A block takes rpb of a token's head rows. Its first wave finds the token's place, its threads the (cos, sin) of the
// pairs once into LDS; then groups of gs lanes (a power of two) take a head row each, a lane up to MU
// pairs of runs of VE elements that turn together (or runs past the turned part). VE 8: the last run of
// a part that is no multiple of 8 begins where it still fits, its first elements being done twice,
// with the same result (a group's lanes are in one wave, which loads a row before it stores it).
// VE 1: parts shorter than 8.
// One token's call is latency (40 heads of 64, f32: 2.7 us; with norm and append 3.5), a long batch is bound by its
// bytes: 4097 tokens of 32 heads of 128, bf16, 14.2 us, 4.7 TB/s read and written; 5003 tokens of 32 query
// and 8 kv heads appended 27.1 us, 4.5 TB/s (a plain copy of 4 GiB: 4.9). Two tokens a block: 14.4 and
// 30 us; elements one at a time where a part is no multiple of 8 (1176 tokens, 118 of 128 turned,
// 28.9 MB): 28 us, in runs 12.7.
template <class A, class C, int VE, bool EVEN>
__global__ void __launch_bounds__(RR_THREADS) k_rope_rows(RopeRows r, RopeTurns rt, PagedView kv, PagedSeqs sq, int rpb,
                                                          int gs) {
  constexpr int MU = VE == 1 ? 4 : 1;
  __shared__ float2 cs[OPS_HD_MAX / 2];
  __shared__ float s_gain[2][OPS_HD_MAX];
  __shared__ RowPlace place;
  const int tid = threadIdx.x, half = rt.half;
  const size_t t = blockIdx.x;
  const int row0 = blockIdx.y * rpb, row1 = min(row0 + rpb, r.n_q + 2 * r.n_kv);
  const int rest = r.hd - 2 * half, nu = (half + VE - 1) / VE, units = nu + (rest + VE - 1) / VE, lane = tid & (gs - 1);

  const double turns = tid < half ? rt.turns[tid] : 0.0;
  if (r.q_norm && tid < r.hd) s_gain[0][tid] = r.q_norm[tid];
  if (r.k_norm && tid < r.hd) s_gain[1][tid] = r.k_norm[tid];
  if (tid < 64) {
    const RowPlace w = row_place(r, kv, sq, t);
    if (tid == 0) place = w;
  }
  __syncthreads();
  const RowPlace w = place;
  if (!w.live) return;  // the whole block
  if (tid < half) {
    const float2 v = cos_sin_turns(w.pos, turns);
    cs[tid] = make_float2(rt.magnitude * v.x, rt.magnitude * v.y);
  }
  __syncthreads();
  // run u's first pair, its first element and how many of its pairs (elements past the turned part) another run has
  const auto pair_of = [&](int u) { return EVEN ? u * VE : min(u * VE, half - VE); };
  const auto rest_of = [&](int u) { return EVEN ? (u - nu) * VE : min((u - nu) * VE, rest - VE); };
  const auto first_of = [&](int u) {
    return u < nu ? (rt.interleaved ? 2 : 1) * pair_of(u) : 2 * half + rest_of(u);
  };
  const auto twice_of = [&](int u) { return EVEN ? 0 : u < nu ? u * VE - pair_of(u) : (u - nu) * VE - rest_of(u); };
  for (int row = row0 + tid / gs; row < row1; row += RR_THREADS / gs) {
    const bool is_q = row < r.n_q, is_k = !is_q && row < r.n_q + r.n_kv;
    if (!is_q && w.base < 0) continue;
    const int head = is_q ? row : is_k ? row - r.n_q : row - r.n_q - r.n_kv;
    const A* x = is_q   ? static_cast<const A*>(r.q) + t * r.q_ts + (size_t)head * r.q_hs
                 : is_k ? static_cast<const A*>(r.k) + t * r.k_ts + (size_t)head * r.hd
                        : static_cast<const A*>(r.v) + t * r.v_ts + (size_t)head * r.hd;
    float a[MU][VE], b[MU][VE];
#pragma unroll
    for (int m = 0; m < MU; ++m) {
      const int u = lane + m * gs, e0 = first_of(u);
#pragma unroll
      for (int j = 0; j < VE; ++j) a[m][j] = b[m][j] = 0.0f;
      if (m * gs >= units) continue;
      if (u < units) load_vec<A, VE>(x + e0, a[m]);
      if (u < nu) load_vec<A, VE>(x + (rt.interleaved ? e0 + VE : e0 + half), b[m]);
    }
    // (in place, a lane stores elements that its neighbour loads too: none may move up past the loads)
    if constexpr (!EVEN) __builtin_amdgcn_wave_barrier();
    A* yq = static_cast<A*>(r.q_out) + t * r.qo_ts + (size_t)head * r.qo_hs;
    C* yc = static_cast<C*>(is_k ? kv.k : kv.v) + w.base + (size_t)head * kv.head_stride;
    if (is_q ? r.q_norm != nullptr : is_k && r.k_norm != nullptr) {
      // rmsnorm over the head: the lanes of the group hold parts of it
      const float* gain = s_gain[is_q ? 0 : 1];
      float ss = 0.0f;
#pragma unroll
      for (int m = 0; m < MU; ++m) {
        const int u = lane + m * gs, twice = twice_of(u);
        const bool flat = rt.interleaved && u < nu;  // a and b are one run of pairs
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          ss += EVEN || j >= (flat ? 2 * twice : twice) ? a[m][j] * a[m][j] : 0.0f;
          ss += EVEN || j >= (flat ? 2 * twice - VE : twice) ? b[m][j] * b[m][j] : 0.0f;
        }
      }
      for (int o = 1; o < gs; o <<= 1) ss += __shfl_xor(ss, o);
      const float scale = 1.0f / sqrtf(ss / (float)r.hd + r.eps);
#pragma unroll
      for (int m = 0; m < MU; ++m) {
        const int u = lane + m * gs, e0 = first_of(u), e1 = rt.interleaved ? e0 + VE : e0 + half;
        if (m * gs >= units) break;
        if (u < units)
#pragma unroll
          for (int j = 0; j < VE; ++j) a[m][j] = a[m][j] * scale * gain[e0 + j];
        if (u < nu)
#pragma unroll
          for (int j = 0; j < VE; ++j) b[m][j] = b[m][j] * scale * gain[e1 + j];
      }
    }
#pragma unroll
    for (int m = 0; m < MU; ++m) {
      const int u = lane + m * gs, e0 = first_of(u), e1 = rt.interleaved ? e0 + VE : e0 + half;
      if (m * gs >= units) break;
      if (u < nu && (is_q || is_k)) {
        const float2* c = cs + pair_of(u);
        if (rt.interleaved && VE > 1) {
          // pairs (0,1), (2,3), ... of the 2·VE elements a, b
#pragma unroll
          for (int j = 0; j < VE; j += 2) {
            const float2 ca = c[j / 2], cb = c[VE / 2 + j / 2];
            const float a0 = a[m][j], a1 = a[m][j + 1], b0 = b[m][j], b1 = b[m][j + 1];
            a[m][j] = a0 * ca.x - a1 * ca.y;
            a[m][j + 1] = a0 * ca.y + a1 * ca.x;
            b[m][j] = b0 * cb.x - b1 * cb.y;
            b[m][j + 1] = b0 * cb.y + b1 * cb.x;
          }
        } else {
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const float a0 = a[m][j], b0 = b[m][j];
            a[m][j] = a0 * c[j].x - b0 * c[j].y;
            b[m][j] = a0 * c[j].y + b0 * c[j].x;
          }
        }
      }
      if (is_q) {
        if (u < units) store_vec<A, VE>(yq + e0, a[m]);
        if (u < nu) store_vec<A, VE>(yq + e1, b[m]);
      } else {
        if (u < units) store_vec<C, VE>(yc + e0, a[m]);
        if (u < nu) store_vec<C, VE>(yc + e1, b[m]);
      }
    }
  }
}

template <class A, class C>
hipError_t rope_rows_of(hipStream_t s, const RopeRows& r, const RopeTurns& t, const PagedView& kv, const PagedSeqs& sq) {
  const int rest = r.hd - 2 * t.half, n_rows = r.n_q + 2 * r.n_kv;
  const bool wide = (t.half == 0 || t.half >= 8) && (rest == 0 || rest >= 8);
  const int ve = wide ? 8 : 1, units = (t.half + ve - 1) / ve + (rest + ve - 1) / ve;
  int gs = 1;
  while (gs < units && gs < 64) gs *= 2;
  const int at_once = RR_THREADS / gs;
  // a token's rows go to several blocks, one turn of the rows each, while all the blocks fit the device at once
  const size_t want = std::max<size_t>(1, std::min<size_t>((n_rows + at_once - 1) / at_once, 2048 / r.T));
  const int rpb = (int)((n_rows + want - 1) / want);
  const dim3 grid((unsigned)r.T, (unsigned)((n_rows + rpb - 1) / rpb));
  if (!wide) BB_LAUNCH((k_rope_rows<A, C, 1, true>), grid, dim3(RR_THREADS), 0, s, r, t, kv, sq, rpb, gs);
  else if (t.half % 8 || rest % 8)
    BB_LAUNCH((k_rope_rows<A, C, 8, false>), grid, dim3(RR_THREADS), 0, s, r, t, kv, sq, rpb, gs);
  else BB_LAUNCH((k_rope_rows<A, C, 8, true>), grid, dim3(RR_THREADS), 0, s, r, t, kv, sq, rpb, gs);
  return hipGetLastError();
}

// f(type of DT a, type of DT b)
template <class F>
hipError_t by_dtypes(int a, int b, F&& f) {
  const auto second = [&](auto x) {
    switch (b) {
      case BB_F32: return f(x, ElemOf<BB_F32>());
      case BB_F16: return f(x, ElemOf<BB_F16>());
      case BB_BF16: return f(x, ElemOf<BB_BF16>());
      default: return hipErrorInvalidValue;
    }
  };
  switch (a) {
    case BB_F32: return second(ElemOf<BB_F32>());
    case BB_F16: return second(ElemOf<BB_F16>());
    case BB_BF16: return second(ElemOf<BB_BF16>());
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_rope_rows(hipStream_t s, int dtype, int cache, const RopeRows& r, const RopeTurns& t,
                            const PagedView& kv, const PagedSeqs& seqs) {
  if (r.T == 0) return hipSuccess;
  if (r.n_kv == 0) cache = dtype;
  return by_dtypes(dtype, cache, [&](auto a, auto c) {
    return rope_rows_of<typename decltype(a)::T, typename decltype(c)::T>(s, r, t, kv, seqs);
  });
}

// ---- attention of one token per sequence ---------------------------------------------------------
//
// out[s][h] = sum_j softmax_j(scale·q·k_j)·v_j in one pass over the keys and values, with the running
// maximum and sum of the softmax. Bound by the cache's bytes: one kv head's keys and values are read
// once for the (up to 16) query heads of a group, and nothing but sums leaves the registers.
//
// 64 sequences of 8192, 32 query on 8 kv heads of 128, f16: 357 to 368 us, 5.8 to 6.0 TB/s; one sequence of 9001, of 64,
// bf16: 13 us, of which 4 are the second launch and 3 pass until the first keys are asked for.
//
// Work. A sequence's positions (from its window's first, rounded down to 32) are cut into units of 128,
// and the units of all (sequence, head group) pairs, in that order, into equal runs, one a block: every
// block reads about the same number of bytes however ragged the batch, with no host knowing a
// length. A pair counts PA_PAIR units more than it has, before its first, for what it costs to begin
// and end it. A block's 4 waves take tiles of KT = 32 positions in turn and are joined in LDS at the end
// of a pair; a pair that lies in several blocks leaves one partial sum each, which k_paged_join adds.
//
// Tiles on the matrix cores, with nothing moved between lanes. Lane l has column (head) n = l%16 and group
// g = l/16. Scores are D[position][head] = K·q^T: A holds 16 positions' rows (lane: row l%16, the group's
// 16-byte pieces), D leaves lane (n, g) the scores of positions 4g..4g+3. Output sums are
// O[element][head] = V^T·p: for B, a lane's own weights (positions 4g..4g+3 of each 16) are already
// where the instruction wants group g's part of the sum, when A's group g holds the values of the
// same positions. So values are loaded row by row, lane m = l%16 an adjacent piece of the row of
// each of its group's positions, and the row index m of instruction i stands for element i of lane
// m's piece; 16-bit pieces are transposed in registers (one byte permute per two values).
//
// Exactness. Scores, weights, maxima and sums are f32. An f32 cache takes f32 matrix instructions. A 16-bit
// cache takes 16-bit ones (an eighth of the time) on its values as they are, with q and the weights
// split into NP 16-bit parts whose products with a cached value are exact in f32: bf16 by truncation (3
// parts are all of an f32; 2 parts, 16 bits and rounded, where q and out are 16-bit themselves), f16
// by rounding (2 parts, 22 bits) after scaling the row of q by the power of two that puts its largest
// in 2^13..2^14 and the weights by 2^14, so that f16's range costs at most 2^-38 of the largest. A part
// that is 0 meets an infinite key as NaN: such scores are taken from the first parts alone.
namespace {

constexpr int PA_WAVES = 4, PA_THREADS = 64 * PA_WAVES;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float NEG_INF = -__builtin_inff();

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// A kv head's G query heads: `split` groups of `hg` (the last may have fewer).
struct PagedPlan {
  int G, split, hg, n_groups, join, unit;  // unit: the logarithm of a unit's positions
  int few;        // blocks that work where pairs are long
  int* chunk;     // [1 + n_seqs + 1]: cost of a block's run, cost of a group in the sequences before each
  float* sums;    // [2·blocks][hg][hd]: of a pair that began in a block before (slot 0), that goes on in the next (1)
  float2* ml;     // [2·blocks][hg]: maximum (base 2), sum of weights
};

__device__ __forceinline__ SeqSpan seq_span(int raw_len, const PagedView& kv, int max_pages, int window, int unit) {
  return span_of(raw_len, kv.page_size, kv.page_slots, max_pages, window, unit);
}

// Four adjacent elements of a row of type dt, at any element's alignment.
template <class T>
__device__ __forceinline__ void store_row(void* p, size_t i, const v4f& x) {
  const float y[4] = {x[0], x[1], x[2], x[3]};
  store_vec<T, 4>(static_cast<T*>(p) + i, y);
}
__device__ __forceinline__ void store_act(void* p, size_t i, int dt, const v4f& x) {
  if (dt == BB_F32) store_row<float>(p, i, x);
  else if (dt == BB_F16) store_row<_Float16>(p, i, x);
  else store_row<__bf16>(p, i, x);
}

// (by value: a bit cast of a vector's element itself reads the vector's first)
__device__ __forceinline__ float as_float(uint32_t a) { return __builtin_bit_cast(float, a); }
__device__ __forceinline__ uint32_t hi_halves(float a, float b) {  // the upper 16 bits of a (low) and b
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ float trunc_bf16(float a) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, a) & 0xffff0000u);
}
// Two values as NP packed 16-bit parts whose sums they are.
template <int CT, int NP>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&w)[NP]) {
  if constexpr (CT == BB_BF16) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (i + 1 == NP && NP < 3) {
        typedef __bf16 v2b __attribute__((ext_vector_type(2)));
        const v2b r = {(__bf16)a, (__bf16)b};
        w[i] = __builtin_bit_cast(uint32_t, r);
      } else {
        w[i] = hi_halves(a, b);
        a = a - trunc_bf16(a);
        b = b - trunc_bf16(b);
      }
    }
  } else {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const v2h r = {(_Float16)a, (_Float16)b};
      w[i] = __builtin_bit_cast(uint32_t, r);
      a = a - (float)r[0];
      b = b - (float)r[1];
    }
  }
}

template <int CT>
__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  if constexpr (CT == BB_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// The four lanes of a column (l, l^16, l^32, l^48): (x, y) -> (lower rows of x and y, upper rows of both).
__device__ __forceinline__ float group_max(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(as_float(a[0]), as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(as_float(b[0]), as_float(b[1]));
}
__device__ __forceinline__ float group_sum(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = as_float(a[0]) + as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return as_float(b[0]) + as_float(b[1]);
}

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the row before's last lane, to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row 1's last lane, to rows 2 and 3
  return x;
}

// A tile's shape: CT the cache's type, HDP the head size (or the next of 64, 128, 256).
template <int CT, int HDP>
struct PaShape {
  static constexpr int SZ = CT == BB_F32 ? 4 : 2;
  static constexpr int KE = 16 / SZ;                     // elements of a 16-byte piece
  static constexpr int NC = HDP / (4 * KE);              // pieces of a key row per lane
  static constexpr int VE = HDP / 16;                    // elements of a value row per lane
  static constexpr int PE = VE < KE ? VE : KE;           // in pieces of PE
  static constexpr int NV = VE / PE;
  static constexpr int KT = CT == BB_F32 ? 16 : 32;      // positions of a tile (registers)
  static constexpr int NT = KT / 16;
};

// One wave's part of a (sequence, head group) pair: running maximum m (base 2), sum l and o[i][r] for element
// (16p + 4g + r)·PE + e, i = p·PE + e, of head n.
// UNI: a page counts as whole 16 positions (slots; up to a third of them empty), whose rows are within 2^31 bytes of
// the first, so that 16 slots have one address the same for the wave. Otherwise every lane finds the
// page of one position and the lanes exchange them. Pages of 24, 64 sequences of 8192 (32 of 4000), UNI
// and not: bf16, 8 kv heads of 64, 211 and 222 us; f16, of 128, 100 and 116 us. Pages of 8, half of
// the slots empty: 300 and 223 us (bf16, 64).
// What is not there or not attended to is loaded as 0 (a weight of 0 times what lies there need not be 0).
template <int CT, int NP, int HDP, bool UNI>
struct PaWave {
  typedef PaShape<CT, HDP> S;
  static constexpr int NT = S::NT, NC = S::NC, NV = S::NV, VE = S::VE, PE = S::PE, KE = S::KE, SZ = S::SZ;
  typedef typename std::conditional<S::PE * S::SZ == 16, v4u, v2u>::type VP;  // a piece of a value row
  const PagedView& kv;
  const int n, g;
  const int* __restrict__ row;  // the sequence's page table
  int head0, heads;  // head0: the first head of the group; heads: how many
  size_t kv_off;     // the kv head's offset in the pool (elements)
  SeqSpan sp;
  v4u q[NP][NC];
  float c;        // what scores are multiplied by where NP is 2
  float m, l;
  v4f o[VE];
  v4u k[NT][NC];
  VP v[4 * NT][NV];
  uint32_t valid;  // bit 4t + r: position 16t + 4g + r of the tile whose values are loaded is attended to
  static constexpr uint32_t ALL = (1u << 4 * NT) - 1;

  __device__ __forceinline__ PaWave(const PagedView& kv_, int lane) : kv(kv_), n(lane & 15), g(lane >> 4) {}

  template <class A>
  __device__ __forceinline__ void load_q(const PagedQuery& pq, int s, float (&x)[NC][KE]) const {
    const size_t at = (size_t)s * pq.q_stride + (size_t)(head0 + min(n, heads - 1)) * kv.hd;
#pragma unroll
    for (int j = 0; j < NC; ++j)
      load_vec<A, KE>(static_cast<const A*>(pq.q) + at + min((4 * j + g) * KE, kv.hd - KE), x[j]);
  }

  __device__ __forceinline__ void start(const PagedQuery& pq, int s) {
    m = NEG_INF;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < VE; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float x[NC][KE];
    if (pq.dt == BB_F32) load_q<float>(pq, s, x);
    else if (pq.dt == BB_F16) load_q<_Float16>(pq, s, x);
    else load_q<__bf16>(pq, s, x);
    // scores are exponents of 2; parts that are all of an f32 take the factor in, two parts only hold q itself
    c = pq.scale * LOG2E;
    const float cq = NP == 2 ? 1.0f : c;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int e = 0; e < KE; ++e) x[j][e] = n < heads && (4 * j + g) * KE < kv.hd ? x[j][e] * cq : 0.0f;
    if constexpr (CT == BB_F16) {
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < KE; ++e) top = fmaxf(top, fabsf(x[j][e]));
      // (0 and what is not finite keep their scale)
      top = group_max(top);
      const int e2 = top > 0.0f && top < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
      c = ldexpf(c, -e2);
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < KE; ++e) x[j][e] = ldexpf(x[j][e], e2);
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if constexpr (CT == BB_F32) {
#pragma unroll
        for (int e = 0; e < KE; ++e) q[0][j][e] = __float_as_uint(x[j][e]);
      } else {
#pragma unroll
        for (int e = 0; e < KE; e += 2) {
          uint32_t w[NP];
          split2<CT, NP>(x[j][e], x[j][e + 1], w);
#pragma unroll
          for (int i = 0; i < NP; ++i) q[i][j][e / 2] = w[i];
        }
      }
    }
  }

  // Where a tile's positions are in the pool (elements; -1: not there, or not attended to): UNI, each 16, the same for
  // the wave, and how many of them from there on the page has; otherwise lane l's is position l % KT's.
  struct Places {
    int key0;
    int64_t at[UNI ? NT : 1];
    int rows[UNI ? NT : 1];
  };
  __device__ __forceinline__ void place(Places& p, int t, int key, int end) const {
    const int i = min(key, sp.len - 1), entry = page_of(kv, i), in = i - entry * kv.page_slots;
    int pg = row[entry];
    if constexpr (UNI) pg = __builtin_amdgcn_readfirstlane(pg);
    const bool there = key < end && (uint32_t)pg < (uint32_t)kv.n_pages;
    const int64_t at = (int64_t)((size_t)(uint32_t)pg * kv.page_stride + (size_t)(uint32_t)in * kv.pos_stride + kv_off);
    p.at[t] = there ? at : -1;
    p.rows[t] = min(16, kv.page_size - in);
  }
  __device__ __forceinline__ Places places(int key0, int end) const {
    Places p;
    p.key0 = key0;
    if constexpr (UNI) {
#pragma unroll
      for (int t = 0; t < NT; ++t) place(p, t, key0 + 16 * t, end);
    } else {
      const int key = key0 + ((n + 16 * g) & (S::KT - 1));
      place(p, 0, key, key >= sp.first ? end : 0);
    }
    return p;
  }

  // UNI: the rows of 16 positions as a buffer that ends with row `rows` - 1 (0 rows: all of it reads as 0).
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* pool, int64_t at, int rows) const {
    const bool there = at >= 0 && rows > 0;
    const char* base = static_cast<const char*>(pool) + (there ? (size_t)at * SZ : 0);
    const uint32_t bytes = there ? (uint32_t)(rows - 1) * stride() + (uint32_t)(kv.hd * SZ) : 0;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, bytes, 0x00027000);
  }
  __device__ __forceinline__ uint32_t stride() const { return (uint32_t)kv.pos_stride * SZ; }

  __device__ __forceinline__ void load_k(const Places& p) {
    if constexpr (UNI) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const auto rows = rows_of(kv.k, p.at[t], p.rows[t]);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          // (pieces past the head: 0, which 0 times what lies there need not be)
          const int d = (4 * j + g) * KE;
          const uint32_t at = d < kv.hd ? (uint32_t)n * stride() + (uint32_t)(d * SZ) : 0x80000000u;
          k[t][j] = __builtin_amdgcn_raw_buffer_load_b128(rows, at, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t at = __shfl(p.at[0], n + 16 * t);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const int d = (4 * j + g) * KE;
          k[t][j] = v4u{0, 0, 0, 0};
          if (at >= 0 && d < kv.hd)
            k[t][j] = *reinterpret_cast<const v4u*>(static_cast<const char*>(kv.k) + (size_t)(at + d) * SZ);
        }
      }
    }
  }

  __device__ __forceinline__ void load_v(const Places& p) {
    valid = 0;
    if constexpr (UNI) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int k0 = p.key0 + 16 * t, skip = max(0, sp.first - k0);
        const int n_rows = min(p.rows[t], sp.len - k0);
        const auto rows = rows_of(kv.v, p.at[t], n_rows);
        if (p.at[t] >= 0) {
          if (skip == 0 && n_rows == 16) {
            valid |= 15u << 4 * t;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) valid |= (4 * g + r >= skip && 4 * g + r < n_rows ? 1u : 0u) << (4 * t + r);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // (pieces past the head end in elements of o that nobody reads; what they fetch counts: 7 sequences with 16
          // heads of 80 fetch 59.9 MB, their keys and values are 31.7)
          const uint32_t at = 4 * g + r < skip ? 0x80000000u : (uint32_t)(4 * g + r) * stride() + (uint32_t)(n * PE * SZ);
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if constexpr (PE * SZ == 16)
              v[4 * t + r][j] = __builtin_amdgcn_raw_buffer_load_b128(rows, at + (uint32_t)(16 * j * PE * SZ), 0, 0);
            else
              v[4 * t + r][j] = __builtin_amdgcn_raw_buffer_load_b64(rows, at + (uint32_t)(16 * j * PE * SZ), 0, 0);
          }
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t at = __shfl(p.at[0], 16 * t + 4 * g + r);
          valid |= (at >= 0 ? 1u : 0u) << (4 * t + r);
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const int d = (16 * j + n) * PE;
            v[4 * t + r][j] = VP{};
            if (at >= 0 && d < kv.hd)
              v[4 * t + r][j] = *reinterpret_cast<const VP*>(static_cast<const char*>(kv.v) + (size_t)(at + d) * SZ);
          }
        }
    }
  }

  template <int PARTS>
  __device__ __forceinline__ void scores(v4f (&x)[NT]) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (CT == BB_F32) {
#pragma unroll
          for (int e = 0; e < KE; ++e)
            x[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(k[t][j][e]), as_float(q[0][j][e]), x[t], 0, 0, 0);
        } else {
#pragma unroll
          for (int i = PARTS - 1; i >= 0; --i) x[t] = mfma16<CT>(k[t][j], q[i][j], x[t]);
        }
      }
  }

  // Scores of the loaded keys, from which the keys' registers are free again.
  __device__ __forceinline__ void score(v4f (&x)[NT]) const {
    scores<NP>(x);
    if constexpr (NP > 1) {
      bool odd = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd |= x[t][r] != x[t][r];
      if (__any(odd)) {
        v4f y[NT];
        scores<1>(y);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (x[t][r] != x[t][r]) x[t][r] = y[t][r];
      }
    }
  }

  // Adds a tile: its scores x and the loaded values.
  __device__ __forceinline__ void add(v4f (&x)[NT]) {
    if constexpr (NP == 2) {
#pragma unroll
      for (int t = 0; t < NT; ++t) x[t] *= c;
    }
    if (__any(valid != ALL)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[t][r] = valid >> (4 * t + r) & 1 ? x[t][r] : NEG_INF;
    }
    float mx = NEG_INF;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[t][r]);
    mx = fmaxf(m, group_max(mx));
    const float ref = mx == NEG_INF ? 0.0f : mx;
    if (__any(mx > m)) {
      const float f = __builtin_amdgcn_exp2f(m - ref);
      l *= f;
#pragma unroll
      for (int i = 0; i < VE; ++i) o[i] *= f;
    }
    m = mx;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[t][r] = __builtin_amdgcn_exp2f(x[t][r] - ref);
        if constexpr (CT == BB_F16) x[t][r] *= 16384.0f;
        l += x[t][r];
      }
    if constexpr (CT == BB_F32) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < VE; ++i)
            o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(v[4 * t + r][i / PE][i % PE]), x[t][r], o[i], 0, 0, 0);
    } else {
      v4u p[NP];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          uint32_t w[NP];
          split2<CT, NP>(x[t][r], x[t][r + 1], w);
#pragma unroll
          for (int i = 0; i < NP; ++i) p[i][2 * t + r / 2] = w[i];
        }
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        v4u a;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          a[w] = __builtin_amdgcn_perm(v[2 * w + 1][i / PE][i % PE / 2], v[2 * w][i / PE][i % PE / 2],
                                       i % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int j = NP - 1; j >= 0; --j) o[i] = mfma16<CT>(a, p[j], o[i]);
      }
    }
  }

  // A whole pair's results from this wave's sums alone.
  __device__ __forceinline__ void finish(const PagedQuery& pq, int s, float up) {
    l = group_sum(l);
    if (n >= heads) return;
    const bool none = m == NEG_INF && l == 0.0f;
    const float f = none ? 0.0f : 1.0f / l;
    const size_t out = (size_t)s * pq.out_stride + (size_t)(head0 + n) * kv.hd;
#pragma unroll
    for (int p = 0; p < NV; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < PE; e += 4) {
          const int d = (16 * p + 4 * g + r) * PE + e, i = p * PE + e;
          if (d < kv.hd) store_act(pq.out, out + d, pq.dt, v4f{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]} * f);
        }
    if (g == 0 && pq.lse)
      pq.lse[(size_t)s * pq.n_heads + head0 + n] = none ? NEG_INF : (m + (__builtin_amdgcn_logf(l) - up)) * LN2;
  }

  // Positions key, key + step, ... below end.
  __device__ __forceinline__ void run(int key, int end, int step) {
    if (key >= end) return;
    Places p = places(key, end);
    load_k(p);
    load_v(p);
    // (The scheduler is held to this order: a load that moved up would need a second set of registers. The
    // last turn's loads are of no pages and touch no memory.)
    for (; key < end; key += step) {
      v4f x[NT];
      p = places(key + step, end);
      __builtin_amdgcn_sched_barrier(0);
      score(x);
      __builtin_amdgcn_sched_barrier(0);
      load_k(p);
      __builtin_amdgcn_sched_barrier(0);
      add(x);
      __builtin_amdgcn_sched_barrier(0);
      load_v(p);
    }
  }
};

// The sequences' costs (units + PA_PAIR), 256 at a time: lane l has sequences c0 + 64i + l, incl[i] the costs from c0
// up to and with its own.
struct SeqScan {
  int c0;
  int len[4], cost[4], incl[4];
  int all;         // of the 256
  __device__ __forceinline__ void load(const int* __restrict__ lens, int n_seqs, const PagedView& kv, int max_pages,
                                       int window, int unit, int lane) {
    all = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) len[i] = c0 + 64 * i < n_seqs ? lens[min(c0 + 64 * i + lane, n_seqs - 1)] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cost[i] = incl[i] = 0;
      if (c0 + 64 * i < n_seqs) {
        cost[i] = c0 + 64 * i + lane < n_seqs ? seq_span(len[i], kv, max_pages, window, unit).units + PA_PAIR : 0;
        incl[i] = all + wave_scan(cost[i]);
        all = __builtin_amdgcn_readlane(incl[i], 63);
      }
    }
  }
};

template <int CT, int NP, int HDP, bool UNI>
__global__ void __launch_bounds__(PA_THREADS, pa_waves(HDP)) k_paged_attn(PagedQuery pq, PagedView kv,
                                                                        const int* __restrict__ table,
                                                                        const int* __restrict__ lens, size_t table_stride,
                                                                        int n_seqs, int max_pages, PagedPlan pl) {
  typedef PaShape<CT, HDP> S;
  constexpr int LD = HDP + 4, ROW4 = HDP / 4;
  extern __shared__ __align__(16) float so[];  // [waves][hg][LD]
  __shared__ float s_m[PA_WAVES][PA_HEADS], s_l[PA_WAVES][PA_HEADS];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);

  // every wave finds the block's run by itself: the total cost, then the sequence in whose cost the run begins
  // (more than 256 sequences are gone through twice)
  int u = 0, end = 0, s = 0, cost = 0, len = 0, lo = 0;
  {
    SeqScan sc;
    sc.c0 = 0;
    int before = 0;
    for (;;) {
      sc.load(lens, n_seqs, kv, max_pages, pq.window, pl.unit, lane);
      if (end == 0) {
        if (pl.join && blockIdx.x == 0 && wv == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (sc.c0 + 64 * i + lane < n_seqs) pl.chunk[2 + sc.c0 + 64 * i + lane] = before + sc.incl[i];
        }
        if (sc.c0 + 256 < n_seqs) {
          before += sc.all;
          sc.c0 += 256;
          continue;
        }
        const int total = (before + sc.all) * pl.n_groups;
        const int chunk = run_cost(before + sc.all, n_seqs, pl.n_groups, (int)gridDim.x, pl.few);
        if (pl.join && blockIdx.x == 0 && tid == 0) {
          pl.chunk[0] = chunk;
          pl.chunk[1] = 0;
        }
        if ((int64_t)blockIdx.x * chunk >= total) return;  // (all work is in the first `grid` blocks)
        u = (int)blockIdx.x * chunk;
        end = min(u + chunk, total);
        before = 0;
        if (sc.c0 > 0) {
          sc.c0 = 0;
          continue;
        }
      }
      if (u < (before + sc.all) * pl.n_groups) break;
      before += sc.all;
      sc.c0 += 256;
    }
    bool found = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (found || sc.c0 + 64 * i >= n_seqs) continue;
      const uint64_t past = __ballot((before + sc.incl[i]) * pl.n_groups > u);
      if (past) {
        const int at = __builtin_ctzll(past);
        found = true;
        s = sc.c0 + 64 * i + at;
        cost = __builtin_amdgcn_readlane(sc.cost[i], at);
        len = __builtin_amdgcn_readlane(sc.len[i], at);
        lo = (before + __builtin_amdgcn_readlane(sc.incl[i], at) - cost) * pl.n_groups;
      }
    }
  }
  int grp = uniform_div(u - lo, cost);
  lo += grp * cost;

  PaWave<CT, NP, HDP, UNI> w(kv, lane);
  const float up = CT == BB_F16 ? 14.0f : 0.0f;
  bool lds_read = false;
  int turn = 0;
  // the run's pairs: group grp of sequence s, whose cost begins at lo
  for (; lo < end; lo += cost, ++grp) {
    if (grp == pl.n_groups) {
      grp = 0;
      ++s;
      len = __builtin_amdgcn_readfirstlane(lens[s]);
      cost = seq_span(len, kv, max_pages, pq.window, pl.unit).units + PA_PAIR;
    }
    const int nu = cost - PA_PAIR;
    const PairPart part = pair_part(u, end, lo, nu);
    const int u0 = part.first, take = part.units;
    if (take <= 0) continue;  // (the run ends before the pair's units)
    const SeqSpan sp = seq_span(len, kv, max_pages, pq.window, pl.unit);
    const bool alone = pair_alone(nu, sp, S::KT, end - u);
    if (alone && (turn++ & (PA_WAVES - 1)) != wv) continue;
    const int kvh = pl.split == 1 ? grp : uniform_div(grp, pl.split), sub = grp - kvh * pl.split;
    w.row = table + (size_t)s * table_stride;
    w.head0 = kvh * pl.G + sub * pl.hg;
    w.heads = min(pl.hg, pl.G - sub * pl.hg);
    w.kv_off = (size_t)kvh * kv.head_stride;
    w.sp = sp;
    w.start(pq, s);
    const int k0 = w.sp.base + (u0 << pl.unit);
    w.run(alone ? k0 : k0 + wv * S::KT, min(k0 + (take << pl.unit), w.sp.len), alone ? S::KT : PA_WAVES * S::KT);
    if (alone) {
      w.finish(pq, s, up);
      continue;
    }

    // the waves' sums together
    if (lds_read) __syncthreads();  // (the pair before is done with LDS)
    lds_read = true;
    const float l_all = group_sum(w.l);
    if (w.g == 0) {
      s_m[wv][w.n] = w.m;
      s_l[wv][w.n] = l_all;
    }
    __syncthreads();
    float top = NEG_INF;
#pragma unroll
    for (int i = 0; i < PA_WAVES; ++i) top = fmaxf(top, s_m[i][w.n]);
    const float f = __builtin_amdgcn_exp2f(w.m - (top == NEG_INF ? 0.0f : top));
    if (w.n < w.heads) {
      float* to = so + (wv * pl.hg + w.n) * LD;
#pragma unroll
      for (int p = 0; p < S::NV; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < S::PE; e += 4)
            *reinterpret_cast<v4f*>(to + (16 * p + 4 * w.g + r) * S::PE + e) =
                v4f{w.o[p * S::PE + e][r], w.o[p * S::PE + e + 1][r], w.o[p * S::PE + e + 2][r],
                    w.o[p * S::PE + e + 3][r]} * f;
    }
    __syncthreads();
    const bool whole = take == nu;
    const size_t slot = partial_slot((int)blockIdx.x, u0 == 0);
    for (int i = tid; i < w.heads * ROW4; i += PA_THREADS) {
      const int h = i / ROW4, d = 4 * (i % ROW4);
      if (d >= kv.hd) continue;
      float mm = NEG_INF, ll = 0.0f;
      v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < PA_WAVES; ++j) mm = fmaxf(mm, s_m[j][h]);
#pragma unroll
      for (int j = 0; j < PA_WAVES; ++j) {
        ll += s_l[j][h] * __builtin_amdgcn_exp2f(s_m[j][h] - (mm == NEG_INF ? 0.0f : mm));
        x += *reinterpret_cast<const v4f*>(so + (j * pl.hg + h) * LD + d);
      }
      if (whole) {
        const bool none = mm == NEG_INF && ll == 0.0f;
        store_act(pq.out, (size_t)s * pq.out_stride + (size_t)(w.head0 + h) * kv.hd + d, pq.dt,
                  x * (none ? 0.0f : 1.0f / ll));
        if (d == 0 && pq.lse)
          pq.lse[(size_t)s * pq.n_heads + w.head0 + h] = none ? NEG_INF : (mm + (__builtin_amdgcn_logf(ll) - up)) * LN2;
      } else {
        *reinterpret_cast<v4f*>(pl.sums + (slot * pl.hg + h) * kv.hd + d) = x;
        if (d == 0) pl.ml[slot * pl.hg + h] = make_float2(mm, ll);
      }
    }
  }
}

// Adds the partial sums of a (sequence, head), PJ_PIECES pieces of 4 elements a block: those of the blocks whose
// runs hold units of it. Threads: a row of PJ_PIECES for every PJ_ROWS-th part, joined in LDS.
constexpr int PJ_THREADS = 256, PJ_PIECES = 8, PJ_ROWS = PJ_THREADS / PJ_PIECES;
__global__ void __launch_bounds__(PJ_THREADS) k_paged_join(PagedQuery pq, int hd, int blocks_of_row, PagedPlan pl,
                                                           float up) {
  __shared__ float s_m[PJ_ROWS], s_l[PJ_ROWS];
  __shared__ v4f s_x[PJ_ROWS][PJ_PIECES];
  const int s = blockIdx.x, grp = blockIdx.y, hh = blockIdx.z / blocks_of_row;
  const int piece = (blockIdx.z - hh * blocks_of_row) * PJ_PIECES + threadIdx.x % PJ_PIECES;
  const int row = threadIdx.x / PJ_PIECES;
  const int chunk = pl.chunk[0], before = pl.chunk[1 + s], cost = pl.chunk[2 + s] - before;
  const PairBlocks blocks = pair_blocks(before * pl.n_groups + grp * cost, cost, chunk);
  const int b0 = blocks.first, b1 = blocks.last;
  if (b0 == b1) return;  // whole in one block
  const int kvh = pl.split == 1 ? grp : grp / pl.split, in = (grp - kvh * pl.split) * pl.hg + hh, h = kvh * pl.G + in;
  if (in >= pl.G) return;  // (the last group of a kv head may have fewer heads)
  const int parts = b1 - b0 + 1;
  float m = NEG_INF, l = 0.0f;
  v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = row; i < parts; i += PJ_ROWS) {
    const size_t at = partial_slot(b0 + i, i == 0) * pl.hg + hh;
    const float2 ml = pl.ml[at];
    const v4f y = *reinterpret_cast<const v4f*>(pl.sums + at * hd + min(4 * piece, hd - 4));
    const float top = fmaxf(m, ml.x), ref = top == NEG_INF ? 0.0f : top;
    const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(ml.x - ref);
    m = top;
    l = l * f0 + ml.y * f1;
    x = x * f0 + y * f1;
  }
  if (threadIdx.x % PJ_PIECES == 0) {
    s_m[row] = m;
    s_l[row] = l;
  }
  s_x[row][threadIdx.x % PJ_PIECES] = x;
  __syncthreads();
  if (threadIdx.x >= PJ_PIECES || 4 * piece >= hd) return;
  m = NEG_INF;
  for (int i = 0; i < PJ_ROWS; ++i) m = fmaxf(m, s_m[i]);
  const float ref = m == NEG_INF ? 0.0f : m;
  l = 0.0f;
  x = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < PJ_ROWS; ++i) {
    const float f = __builtin_amdgcn_exp2f(s_m[i] - ref);
    l += s_l[i] * f;
    x += s_x[i][threadIdx.x] * f;
  }
  const bool none = m == NEG_INF && l == 0.0f;
  store_act(pq.out, (size_t)s * pq.out_stride + (size_t)h * hd + 4 * piece, pq.dt, x * (none ? 0.0f : 1.0f / l));
  if (piece == 0 && pq.lse)
    pq.lse[(size_t)s * pq.n_heads + h] = none ? NEG_INF : (m + (__builtin_amdgcn_logf(l) - up)) * LN2;
}

}  // namespace

bool paged_attn_fits(int n_seqs, int n_heads, int n_kv, size_t cap) {
  return head_groups(n_heads, n_kv).fits(n_seqs, cap);
}

void PagedView::set_slots(int n) {
  const SlotDivision d = slot_division(n);
  page_slots = n;
  page_mul = d.mul;
  page_shift = d.shift;
}

size_t paged_attn_ws(int n_cu, int n_seqs, int n_heads, int n_kv, int hd) {
  const size_t slots = 2 * (size_t)blocks_at_once(n_cu, hd) * head_groups(n_heads, n_kv).hg;
  return slots * ((size_t)hd * 4 + sizeof(float2)) + ((size_t)n_seqs + 2) * 4;
}

hipError_t launch_paged_attn(hipStream_t st, int n_cu, int cache, const PagedQuery& q, const PagedView& pool,
                             const PagedSeqs& sq) {
  if (sq.n_seqs == 0) return hipSuccess;
  const HeadGroups g = head_groups(q.n_heads, pool.n_kv);
  const PagedCut cut = paged_cut(n_cu, sq.n_seqs, g.n_groups, pool.page_size, pool.pos_stride, sq.max_pages, q.window,
                                 pool.hd, cache == BB_F32 ? 4 : 2);
  const bool uni = cut.uni;
  PagedView kv = pool;
  if (uni) kv.set_slots(cut.slots);
  PagedPlan pl{g.G, g.split, g.hg, g.n_groups, cut.join, cut.unit, cut.few, nullptr, nullptr, nullptr};
  const size_t slots = 2 * (size_t)blocks_at_once(n_cu, kv.hd) * pl.hg;
  pl.sums = static_cast<float*>(q.ws);
  pl.ml = reinterpret_cast<float2*>(pl.sums + slots * kv.hd);
  pl.chunk = reinterpret_cast<int*>(pl.ml + slots);
  const unsigned blocks = (unsigned)cut.blocks;
  const int cls = pa_class(kv.hd);
  const size_t lds = (size_t)PA_WAVES * pl.hg * (cls + 4) * 4;
#define BB_PA(ct, np, hdp)                                                                                     \
  do {                                                                                                         \
    if (uni)                                                                                                   \
      BB_LAUNCH((k_paged_attn<ct, np, hdp, true>), dim3(blocks), dim3(PA_THREADS), lds, st, q, kv, sq.table,   \
                sq.lens, sq.table_stride, sq.n_seqs, sq.max_pages, pl);                                        \
    else                                                                                                       \
      BB_LAUNCH((k_paged_attn<ct, np, hdp, false>), dim3(blocks), dim3(PA_THREADS), lds, st, q, kv, sq.table,  \
                sq.lens, sq.table_stride, sq.n_seqs, sq.max_pages, pl);                                        \
  } while (0)
#define BB_PA_HD(ct, np)             \
  do {                               \
    if (cls == 64) BB_PA(ct, np, 64); \
    else if (cls == 128) BB_PA(ct, np, 128); \
    else BB_PA(ct, np, 256);         \
  } while (0)
  if (cache == BB_F32) BB_PA_HD(BB_F32, 1);
  else if (cache == BB_F16) BB_PA_HD(BB_F16, 2);
  else if (q.dt == BB_F32) BB_PA_HD(BB_BF16, 3);
  else BB_PA_HD(BB_BF16, 2);
#undef BB_PA_HD
#undef BB_PA
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !pl.join) return e;
  const int blocks_of_row = (kv.hd + 4 * PJ_PIECES - 1) / (4 * PJ_PIECES);
  BB_LAUNCH(k_paged_join, dim3(sq.n_seqs, pl.n_groups, pl.hg * blocks_of_row), dim3(PJ_THREADS), 0, st, q, kv.hd,
            blocks_of_row, pl, cache == BB_F16 ? 14.0f : 0.0f);
  return hipGetLastError();
}

}  // namespace bb
