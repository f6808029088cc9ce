// bb_paged_prompt.hip — attention of several new tokens per sequence over a paged cache: prompts, chunks of
// them, drafts to verify (include/bebelm_moe.h states the operator). The reference has no counterpart.
#include <algorithm>
#include "bb_paged4.h"
#include "bb_paged_device.h"
#include "bb_prompt_plan.h"

namespace bb {

namespace {

constexpr int PP_THREADS = 256;
// Weights go up to 2^SLACK, as f16 to 2^(SLACK + F16_UP) = 2^14, whose range then costs at most 2^-33 of the largest.
constexpr float SLACK = 6.0f, F16_UP = 8.0f;
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

// A block's shape. CT: the type that tiles have in LDS; WR waves along the rows (32 each), 4 / WR along the keys.
template <int CT, int NQ, int NP, int HDP, int WR, bool KV4>
struct PpShape {
  static constexpr int SZ = CT == BB_F32 ? 4 : 2;
  static constexpr int WK = 4 / WR, BM = 32 * WR;
  static constexpr int BN = WK > 1 || HDP * SZ >= 1024 ? 32 : 64;  // keys of a wave's tile
  static constexpr int KT = WK * BN;                               // keys of the block's
  static constexpr int NT = BN / 32;
  // Rows in LDS: 16-byte pieces, of which row r has piece u at place u ^ k_swap(r) (keys) or u ^ v_swap(r) (values).
  // Keys are read a piece of 16 rows at once, 16-bit values 4 pieces of 4 rows, f32 values 8 pieces of
  // rows 4 apart: each time all banks.
  static constexpr int ROW = HDP * SZ, PPR = ROW / 16;
  __device__ static __forceinline__ int k_swap(int r) { return PPR == 8 ? r >> 1 & 7 : r & 15; }
  __device__ static __forceinline__ int v_swap(int r) {
    return SZ == 4 ? (r >> 2 & 1) << 3 : PPR == 8 ? (r >> 1 & 1) << 2 : (r & 3) << 2;
  }
  static constexpr int BUF = 2 * KT * ROW;
  static constexpr int NBUF = 2 * BUF <= 158 * 1024 ? 2 : 1;
  static constexpr int LD = HDP + 4;                                        // a row of the waves' sums, in the same place
  static constexpr int SUMS = WK > 1 ? 4 * 32 * (LD * 4 + 8) : 0;
  static constexpr int LDS = NBUF * BUF > SUMS ? NBUF * BUF : SUMS;
  static constexpr int RPW = KT / 4;  // rows a wave brings
  // pieces of 16 bytes in LDS that a lane brings of keys (and of values); of a 4-bit cache, units of UE elements
  static constexpr int NPC = RPW * PPR / 64;
  static constexpr int UE = RPW * HDP / 64 < 32 ? RPW * HDP / 64 : 32, UPR = HDP / UE, NU = RPW * UPR / 64;
  static constexpr int QW = CT == BB_F32 ? HDP / 2 : NQ * HDP / 4;  // registers of the query rows
  static constexpr int REGS = HDP / 2 + QW + 16 * NT + (CT == BB_F32 ? 0 : 8 * NP * NT) +
                              (KV4 ? 2 * NU * (UE / 8 + 1) : 0);
  static constexpr int WAVES = REGS <= 208 && LDS <= 79 * 1024 ? 2 : 1;  // of a SIMD
};

__device__ __attribute__((aligned(16))) uint32_t g_zeros[4];
// 16 bytes of every lane from its own address to lds + 16·lane.
__device__ __forceinline__ void to_lds(const char* from, char* lds) {
  typedef __attribute__((address_space(1))) const uint32_t* global_u32;
  typedef __attribute__((address_space(3))) uint32_t* lds_u32;
  __builtin_amdgcn_global_load_lds((global_u32)(from), (lds_u32)(lds), 16, 0, 0);
}
// All of a wave's loads into LDS are there, for the waves behind the barrier that follows.
__device__ __forceinline__ void landed() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

__device__ __forceinline__ float half_max(float x) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(as_float(b[0]), as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return as_float(b[0]) + as_float(b[1]);
}

template <int CT>
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
  if constexpr (CT == BB_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Two 16-bit elements: those that are not finite, as 1s of the type (0: finite), and the others as they are.
template <int CT>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  constexpr uint32_t EXP = CT == BB_BF16 ? 0x7f80u : 0x7c00u, ONE = CT == BB_BF16 ? 0x3f80u : 0x3c00u;
  return ((w & EXP) == EXP ? ONE : 0u) | ((w & EXP << 16) == EXP << 16 ? ONE << 16 : 0u);
}
__device__ __forceinline__ uint32_t fine_halves(uint32_t w, uint32_t odd) {
  return w & ~((odd & 0xffffu ? 0xffffu : 0u) | (odd >> 16 ? 0xffff0000u : 0u));
}

// tanh, within a few units in the last place: up to 0.6 a quotient of polynomials (the continued fraction
// y / (1 + y^2 / (3 + y^2 / (5 + y^2 / (7 + y^2 / 9)))), off by less than 1e-9 there), then (e - 1) / (e + 1), e = exp(2|y|).
__device__ __forceinline__ float tanh_of(float y) {
  const float a = fabsf(y), z = y * y;
  const float e = __builtin_amdgcn_exp2f((a > 15.0f ? 15.0f : a) * (2.0f * LOG2E));
  const bool small = a < 0.6f;
  float n0 = a * (fmaf(z, 105.0f + z, 945.0f)), d0 = fmaf(z, fmaf(z, 15.0f, 420.0f), 945.0f), n1 = e - 1.0f, d1 = e + 1.0f;
  asm("" : "+v"(n0), "+v"(d0), "+v"(n1), "+v"(d1));  // (both in line: a branch each would cost more)
  const float num = small ? n0 : n1, den = small ? d0 : d1;
  return copysignf(num * __builtin_amdgcn_rcpf(den), y);
}

// The work of a launch: n_tiles (or fewer) tiles of rows, each for n_kv heads, its keys in up to `parts` parts of
// `least` tiles and more. The sums of parts, and for each tile and head (parts used, first row, rows and first token of
// its sequence), where there may be several.
struct PromptPlan {
  int G, n_tiles, n_kv, parts, least;
  float* sums;   // [tile][kv head][part][row][hd]
  float2* ml;    // [tile][kv head][part][row]: maximum (base 2), sum of weights
  int4* places;  // [tile][kv head]
};

template <int CT, int NQ, int NP, int HDP, int WR, bool KV4>
struct PpWave {
  typedef PpShape<CT, NQ, NP, HDP, WR, KV4> S;
  static constexpr int NT = S::NT, SZ = S::SZ;
  static constexpr bool F16 = CT == BB_F16;
  const PagedView& kv;
  const PromptQuery& pq;
  const int lane, col, half, wv, wr, wk;  // col: the wave's row that is the lane's
  const int* __restrict__ row;            // the sequence's page table
  size_t kv_off;
  int len, prefix;
  int i, lo;                  // the row's token's index, and what it sees first
  int i0, i1, lo1;            // of the wave's first row, of its last
  float c, slope;             // what scores are multiplied by; the bias of a step of distance (base 2)
  float m, l;
  v4u q[NQ][HDP / 16];
  v4f qf[CT == BB_F32 ? HDP / 8 : 1];
  v16f o[HDP / 32];
  uint32_t ck[KV4 ? S::NU * S::UE / 8 : 1], cv[KV4 ? S::NU * S::UE / 8 : 1], hk[KV4 ? S::NU : 1], hv[KV4 ? S::NU : 1];
  int page, in;               // of the row that the lane finds for its wave (page -1: not there)

  __device__ __forceinline__ PpWave(const PagedView& kv_, const PromptQuery& pq_, int tid)
      : kv(kv_), pq(pq_), lane(tid & 63), col(tid & 31), half((tid >> 5) & 1),
        wv(__builtin_amdgcn_readfirstlane(tid >> 6)), wr(wv / S::WK), wk(wv % S::WK) {}

  template <class A>
  __device__ __forceinline__ void load_q(size_t at, float sign) {
    const A* p = static_cast<const A*>(pq.q) + at;
    if constexpr (CT == BB_F32) {
#pragma unroll
      for (int j = 0; j < HDP / 8; ++j) {
        float x[4];
        const int d = 8 * j + 4 * half;
        load_vec<A, 4>(p + min(d, kv.hd - 4), x);
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[j][e] = d < kv.hd ? x[e] * sign : 0.0f;
      }
    } else {
      int up = 0;
      if constexpr (F16) {
        // the power of two that puts the row's largest in 2^13..2^14 (0 and what is not finite keep their scale)
        float top = 0.0f;
#pragma unroll 4
        for (int j = 0; j < HDP / 16; ++j) {
          float x[8];
          load_vec<A, 8>(p + min(16 * j + 8 * half, kv.hd - 8), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
        }
        top = half_max(top);
        up = top > 0.0f && top < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
        c = ldexpf(c, -up);
      }
#pragma unroll
      for (int j = 0; j < HDP / 16; ++j) {
        float x[8];
        const int d = 16 * j + 8 * half;
        load_vec<A, 8>(p + min(d, kv.hd - 8), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = d < kv.hd ? F16 ? ldexpf(x[e] * sign, up) : x[e] * sign : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          uint32_t w[NQ];
          split2<CT, NQ>(x[e], x[e + 1], w);
#pragma unroll
          for (int k = 0; k < NQ; ++k) q[k][j][e / 2] = w[k];
        }
      }
    }
  }

  // The page of tile `t`'s row that this lane looks up: lane r of the wave row r (mod RPW).
  __device__ __forceinline__ void find(int t) {
    const int key = t * S::KT + wv * S::RPW + (lane & (S::RPW - 1));
    page = -1;
    in = 0;
    if (key < len) {
      const int entry = page_of(kv, key);
      in = key - entry * kv.page_size;
      page = row[entry];
    }
  }

  // Asks for the rows found: 4-bit ones into registers, others straight into the tiles at `lds`, 1024 bytes an
  // instruction, each lane a piece (zeros where nothing is). Returns which of the wave's rows are there.
  __device__ __forceinline__ uint32_t load(char* lds) {
    const bool there = (uint32_t)page < (uint32_t)kv.n_pages;
    const uint32_t ok = (uint32_t)__ballot(there) & (~0u >> (32 - S::RPW));
    if constexpr (KV4) {
      const size_t at = there ? (size_t)(uint32_t)page * kv.page_stride + kv_off : 0;
      const uint32_t alo = (uint32_t)at, ahi = (uint32_t)(at >> 32);
      const int pos = there ? in : -1;
#pragma unroll
      for (int p = 0; p < S::NU; ++p) {
        const int e = p * 64 + lane, r = e / S::UPR, u = e % S::UPR, d = u * S::UE;
        const size_t base = (size_t)__shfl((int)ahi, r) << 32 | (uint32_t)__shfl((int)alo, r);
        const int rp = __shfl(pos, r);
        hk[p] = hv[p] = 0;
#pragma unroll
        for (int w = 0; w < S::UE / 8; ++w) ck[p * S::UE / 8 + w] = cv[p * S::UE / 8 + w] = 0;
        if (rp >= 0 && d < kv.hd) {
          const size_t codes = base + (size_t)(uint32_t)(rp * (kv.hd / 2) + d / 2);
          const size_t head = base + (size_t)(uint32_t)kv4_head_at(kv, rp, d / 32);
          load_words<S::UE / 8>(static_cast<const char*>(kv.k) + codes, ck + p * S::UE / 8);
          load_words<S::UE / 8>(static_cast<const char*>(kv.v) + codes, cv + p * S::UE / 8);
          hk[p] = *reinterpret_cast<const uint16_t*>(static_cast<const char*>(kv.k) + head);
          hv[p] = *reinterpret_cast<const uint16_t*>(static_cast<const char*>(kv.v) + head);
        }
      }
    } else {
      const int64_t at = there ? (int64_t)((size_t)(uint32_t)page * kv.page_stride +
                                           (size_t)(uint32_t)in * kv.pos_stride + kv_off)
                               : -1;
      const uint32_t alo = (uint32_t)at, ahi = (uint32_t)(at >> 32);
      char* lk = lds + wv * S::RPW * S::ROW;
#pragma unroll
      for (int p = 0; p < S::NPC; ++p) {
        const int e = p * 64 + lane, r = e / S::PPR, u = e % S::PPR, rr = wv * S::RPW + r;
        const int64_t base = (int64_t)((uint64_t)(uint32_t)__shfl((int)ahi, r) << 32 | (uint32_t)__shfl((int)alo, r));
        const int dk = (u ^ S::k_swap(rr)) * (16 / SZ), dv = (u ^ S::v_swap(rr)) * (16 / SZ);
        const auto from = [&](const void* pool, int d) {
          uint64_t a = reinterpret_cast<uint64_t>(pool) + (uint64_t)(base + d) * SZ;
          asm("" : "+v"(a));  // (a select, no branch)
          return reinterpret_cast<const char*>(base >= 0 && d < kv.hd ? a : reinterpret_cast<uint64_t>(g_zeros));
        };
        to_lds(from(kv.k, dk), lk + p * 1024);
        to_lds(from(kv.v, dv), lk + S::KT * S::ROW + p * 1024);
      }
    }
    return ok;
  }

  // Puts 4-bit rows into the tiles, as the f16 values they stand for.
  __device__ __forceinline__ void put(char* lds) const {
    if constexpr (KV4) {
#pragma unroll
      for (int p = 0; p < S::NU; ++p) {
        const int e = p * 64 + lane, r = wv * S::RPW + e / S::UPR, u = e % S::UPR;
        const Kv4Block bk(hk[p]), bv(hv[p]);
        char* lk = lds + r * S::ROW;
#pragma unroll
        for (int w = 0; w < S::UE / 8; ++w) {
          const int piece = u * (S::UE / 8) + w;
          *reinterpret_cast<v4u*>(lk + (piece ^ S::k_swap(r)) * 16) = bk.natural(ck[p * S::UE / 8 + w]);
          *reinterpret_cast<v4u*>(lk + S::KT * S::ROW + (piece ^ S::v_swap(r)) * 16) = bv.natural(cv[p * S::UE / 8 + w]);
        }
      }
    }
  }

  // Scores of 32 keys for 32 rows: register e of lane (row, half) is key 8(e / 4) + 4·half + e % 4.
  template <int PARTS>
  __device__ __forceinline__ void scores(const char* lk, v16f (&x)[NT]) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[t][e] = 0.0f;
      const int r = wk * S::BN + 32 * t + col;
      const char* at = lk + r * S::ROW;
      const int swap = S::k_swap(r);
      if constexpr (CT == BB_F32) {
#pragma unroll
        for (int j = 0; j < HDP / 8; ++j) {
          const v4f a = *reinterpret_cast<const v4f*>(at + ((2 * j + half) ^ swap) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], qf[j][e], x[t], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < HDP / 16; ++j) {
          const v4u a = *reinterpret_cast<const v4u*>(at + ((2 * j + half) ^ swap) * 16);
#pragma unroll
          for (int k = PARTS - 1; k >= 0; --k) x[t] = mfma32<CT>(a, q[k][j], x[t]);
        }
      }
    }
  }

  // Elements 32·dt + lane % 32 of the values at the keys whose weights are registers 8s..8s+7 of a tile (16-bit types).
  __device__ __forceinline__ v4u values(const char* lv, int t, int s, int dt) const {
    const int r = wk * S::BN + 32 * t + 16 * s + 4 * half + (lane & 15) / 4;
    const int piece = 4 * dt + (lane & 16) / 8 + (lane & 2) / 2;
    const char* at = lv + r * S::ROW + (piece ^ S::v_swap(r)) * 16 + (lane & 1) * 8;
    typedef __attribute__((address_space(3))) v4s* lds_v4s;
    const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(at));
    const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(at + 8 * S::ROW));
    const v2u x = __builtin_bit_cast(v2u, a), y = __builtin_bit_cast(v2u, b);
    return v4u{x[0], x[1], y[0], y[1]};
  }
  // (the same of an f32 cache: at the key of register e)
  __device__ __forceinline__ float value(const char* lv, int t, int e, int dt) const {
    const int r = wk * S::BN + 32 * t + 8 * (e / 4) + 4 * half + e % 4;
    return *reinterpret_cast<const float*>(lv + r * S::ROW + ((8 * dt + col / 4) ^ S::v_swap(r)) * 16 + col % 4 * 4);
  }

  // Which of 32 keys from j0 on the row sees, of those in `ok`: the bits of the lane's registers e at 8(e / 4) + e % 4.
  __device__ __forceinline__ uint32_t seen(int j0, uint32_t ok) const {
    const auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; };  // keys 0..n-1
    return ((below(i + 1 - j0) & ~below(lo - j0)) | below(prefix - j0)) & ok;
  }

  // One tile: keys from j0 on, `ok` those that are there. Values that are not finite reach the rows that see them and no
  // others: where a tile is not seen whole by all rows of the wave, its values are looked at first, and where one is
  // not finite it counts as 0 in the sums and makes NaN of those of the rows that see it.
  __device__ __forceinline__ void tile(const char* lk, const char* lv, int j0, uint32_t ok0, uint32_t ok1) {
    if (j0 >= prefix && (j0 > i1 || j0 + S::BN <= first_seen(i0, pq.window))) return;
    v16f x[NT];
    scores<NQ>(lk, x);
    if constexpr (NQ > 1) {
      // a part of 0 meets an infinite key as NaN: such scores are taken from the first parts alone
      bool odd = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) odd |= x[t][e] != x[t][e];
      if (__any(odd)) {
        v16f y[NT];
        scores<1>(lk, y);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (x[t][e] != x[t][e]) x[t][e] = y[t][e];
      }
    }
    const bool there = ok0 == ~0u && (NT == 1 || ok1 == ~0u);
    const bool whole = there && ((j0 + S::BN - 1 <= i0 && j0 >= lo1) || j0 + S::BN <= prefix);
    float by = c;
    if (pq.cap > 0.0f) {
      by = 1.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] = (pq.cap * LOG2E) * tanh_of(x[t][e] * c);
    } else if (pq.slopes) {
      by = 1.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] *= c;
    }
    if (pq.slopes) {
      const float away = (float)(i - j0 - 4 * half);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[t][e] = fmaf(-slope, fabsf(away - (float)(32 * t + 8 * (e / 4) + e % 4)), x[t][e]);
    }
    if (!whole) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t see = seen(j0 + 32 * t, t ? ok1 : ok0) >> 4 * half;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] = see >> (8 * (e / 4) + e % 4) & 1 ? x[t][e] : NEG_INF;
      }
    }
    float mx = NEG_INF;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, x[t][e]);
    mx = half_max(mx) * by;
    // (m stays until a score is SLACK past it: the sums are as exact, and seldom multiplied)
    const bool past = mx > m + SLACK;
    mx = past ? mx : m;
    const float ref = mx == NEG_INF ? 0.0f : mx;
    if (__any(past)) {
      const float f = __builtin_amdgcn_exp2f(m - ref);
      l *= f;
#pragma unroll
      for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= f;
    }
    m = mx;
    const float less = F16 ? F16_UP - ref : -ref;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[t][e] = __builtin_amdgcn_exp2f(fmaf(x[t][e], by, less));
        l += x[t][e];
      }
    if (whole || !values_odd(lv)) {
      add<false>(lv, x);
    } else {
      add<true>(lv, x);
      mark(lv, j0, ok0, ok1);
    }
  }

  __device__ __forceinline__ bool values_odd(const char* lv) const {
    bool odd = false;
#pragma unroll 1
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int d = 0; d < HDP / 32; ++d) {
        if constexpr (CT == BB_F32) {
#pragma unroll
          for (int e = 0; e < 16; ++e) odd |= !(fabsf(value(lv, t, e, d)) < __builtin_inff());
        } else {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const v4u a = values(lv, t, s, d);
#pragma unroll
            for (int w = 0; w < 4; ++w) odd |= odd_halves<CT>(a[w]) != 0;
          }
        }
      }
    return __any(odd);
  }

  // The values times their weights x (ODD: those that are finite).
  template <bool ODD>
  __device__ __forceinline__ void add(const char* lv, const v16f (&x)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (CT == BB_F32) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int d = 0; d < HDP / 32; ++d) {
            float a = value(lv, t, e, d);
            if (ODD) a = fabsf(a) < __builtin_inff() ? a : 0.0f;
            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[t][e], o[d], 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          v4u p[NP];
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            uint32_t w[NP];
            split2<CT, NP>(x[t][8 * s + e], x[t][8 * s + e + 1], w);
#pragma unroll
            for (int k = 0; k < NP; ++k) p[k][e / 2] = w[k];
          }
#pragma unroll
          for (int d = 0; d < HDP / 32; ++d) {
            v4u a = values(lv, t, s, d);
            if constexpr (ODD) {
#pragma unroll
              for (int w = 0; w < 4; ++w) a[w] = fine_halves(a[w], odd_halves<CT>(a[w]));
            }
#pragma unroll
            for (int k = NP - 1; k >= 0; --k) o[d] = mfma32<CT>(a, p[k], o[d]);
          }
        }
      }
    }
  }

  // NaN for the sums that a value which is not finite belongs to: how many each row sees of them, by the same products.
  __device__ __forceinline__ void mark(const char* lv, int j0, uint32_t ok0, uint32_t ok1) {
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d) {
      v16f n;
#pragma unroll
      for (int e = 0; e < 16; ++e) n[e] = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t see = seen(j0 + 32 * t, t ? ok1 : ok0) >> 4 * half;
        const auto bit = [&](int e) { return see >> (8 * (e / 4) + e % 4) & 1; };
        if constexpr (CT == BB_F32) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float a = fabsf(value(lv, t, e, d)) < __builtin_inff() ? 0.0f : 1.0f;
            n = __builtin_amdgcn_mfma_f32_32x32x2f32(a, (float)bit(e), n, 0, 0, 0);
          }
        } else {
          constexpr uint32_t ONE = CT == BB_BF16 ? 0x3f80u : 0x3c00u;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            v4u a = values(lv, t, s, d), p;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              a[w] = odd_halves<CT>(a[w]);
              p[w] = (bit(8 * s + 2 * w) ? ONE : 0u) | (bit(8 * s + 2 * w + 1) ? ONE << 16 : 0u);
            }
            n = mfma32<CT>(a, p, n);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = n[e] > 0.0f ? __builtin_nanf("") : o[d][e];
    }
  }
};

template <int CT, int NQ, int NP, int HDP, int WR, bool KV4>
__global__ void __launch_bounds__(PP_THREADS, (PpShape<CT, NQ, NP, HDP, WR, KV4>::WAVES))
    k_paged_prompt(PromptQuery pq, PagedView kv, PagedSeqs sq, PromptPlan pl) {
  typedef PpShape<CT, NQ, NP, HDP, WR, KV4> S;
  __shared__ __align__(1024) char s_tiles[S::LDS];
  __shared__ uint32_t s_ok[2][4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kvh = blockIdx.x % pl.n_kv, rest = blockIdx.x / pl.n_kv;
  const int part = rest % pl.parts, g = rest / pl.parts;

  // the sequence whose tile this is (every wave by itself)
  int s = -1, it = 0, a = 0, n = 0;
  for (int b = 0, before = 0; b < sq.n_seqs; b += 64) {
    const int si = min(b + lane, sq.n_seqs - 1);
    TokenSpan sp{si, 1};
    if (pq.seq_start) sp = token_span(pq.seq_start[si], pq.seq_start[si + 1], pq.n_tokens);
    const int tiles = b + lane < sq.n_seqs ? row_tiles(sp.n, pl.G, S::BM) : 0;
    const int incl = wave_scan(tiles);
    const uint64_t past = __ballot(before + incl > g);
    if (past) {
      const int at = __builtin_ctzll(past);
      s = b + at;
      const int mine = __builtin_amdgcn_readlane(tiles, at);
      // the tiles that see most first
      it = mine - 1 - (g - before - (__builtin_amdgcn_readlane(incl, at) - mine));
      a = __builtin_amdgcn_readlane(sp.first, at);
      n = __builtin_amdgcn_readlane(sp.n, at);
      break;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  if (s < 0) {  // (the whole block)
    if (part == 0 && tid == 0 && pl.parts > 1) pl.places[g * pl.n_kv + kvh] = make_int4(0, 0, 0, 0);
    return;
  }

  PpWave<CT, NQ, NP, HDP, WR, KV4> w(kv, pq, tid);
  const int raw = sq.lens[s], end = pq.seq_start ? pq.seq_start[s + 1] : s + 1;
  w.len = min(max(raw, 0), sq.max_pages * kv.page_size);
  w.prefix = pq.prefix ? min(max(pq.prefix[s], 0), w.len) : 0;
  w.row = sq.table + (size_t)s * sq.table_stride;
  w.kv_off = (size_t)kvh * kv.head_stride;
  const int rows = n * pl.G, r0 = it * S::BM;
  const auto index_of = [&](int r) { return token_index(raw, end, a + r / pl.G); };
  const KeyTiles kt =
      key_tiles(index_of(r0), index_of(min(r0 + S::BM, rows) - 1), w.len, w.prefix, pq.window, S::KT);
  const KeyParts kp = key_parts(kt.n, pl.parts, pl.least);
  if (part >= kp.used) return;
  if (part == 0 && tid == 0 && pl.parts > 1) pl.places[g * pl.n_kv + kvh] = make_int4(kp.used, r0, rows, a);
  const int u0 = part * kp.per, u1 = min(kt.n, u0 + kp.per);

  const int mine = r0 + 32 * w.wr + w.col, r = min(mine, rows - 1);
  const int t = a + r / pl.G, head = kvh * pl.G + r % pl.G;
  w.i = token_index(raw, end, t);
  w.lo = first_seen(w.i, pq.window);
  w.i0 = __builtin_amdgcn_readlane(w.i, 0);
  w.i1 = __builtin_amdgcn_readlane(w.i, 31);
  w.lo1 = __builtin_amdgcn_readlane(w.lo, 31);
  w.slope = pq.slopes ? pq.slopes[head] * LOG2E : 0.0f;
  w.c = pq.cap > 0.0f ? fabsf(pq.scale) / pq.cap : fabsf(pq.scale) * LOG2E;
  w.m = NEG_INF;
  w.l = 0.0f;
#pragma unroll
  for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) w.o[d][e] = 0.0f;
  {
    const size_t at = (size_t)t * pq.q_stride + (size_t)head * kv.hd;
    const float sign = pq.scale < 0.0f ? -1.0f : 1.0f;
    if (pq.dt == BB_F32) w.template load_q<float>(at, sign);
    else if (pq.dt == BB_F16) w.template load_q<_Float16>(at, sign);
    else w.template load_q<__bf16>(at, sign);
    w.c = fmaxf(w.c, 1e-37f);  // (0 times an infinite score would be NaN)
  }

  if (u0 < u1) {
    w.find(kt.at(u0));
    uint32_t ok = w.load(s_tiles);
    if (u0 + 1 < u1) w.find(kt.at(u0 + 1));
    w.put(s_tiles);
    if (lane == 0) s_ok[0][w.wv] = ok;
    landed();
    __syncthreads();
    for (int u = u0; u < u1; ++u) {
      const int buf = S::NBUF == 2 ? (u - u0) & 1 : 0, flag = (u - u0) & 1;
      const char* tiles = s_tiles + buf * S::BUF;
      char* next = s_tiles + (S::NBUF == 2 ? buf ^ 1 : 0) * S::BUF;
      // (one buffer: other tiles than 4-bit ones come when all waves are done with this one)
      constexpr bool EARLY = S::NBUF == 2 || KV4;
      if (EARLY && u + 1 < u1) {
        ok = w.load(next);
        if (u + 2 < u1) w.find(kt.at(u + 2));
      }
      uint32_t ok0, ok1 = ~0u;
      if constexpr (S::RPW == 32) {
        ok0 = s_ok[flag][w.wk];
      } else if constexpr (S::WK == 1 && S::RPW == 16) {
        ok0 = s_ok[flag][0] | s_ok[flag][1] << 16;
        ok1 = s_ok[flag][2] | s_ok[flag][3] << 16;
      } else if constexpr (S::WK == 2) {
        ok0 = s_ok[flag][2 * w.wk] | s_ok[flag][2 * w.wk + 1] << 16;
      } else {
        ok0 = s_ok[flag][0] | s_ok[flag][1] << 8 | s_ok[flag][2] << 16 | s_ok[flag][3] << 24;
      }
      ok0 = __builtin_amdgcn_readfirstlane(ok0);
      ok1 = __builtin_amdgcn_readfirstlane(ok1);
      w.tile(tiles, tiles + S::KT * S::ROW, kt.at(u) * S::KT + w.wk * S::BN, ok0, ok1);
      if (u + 1 < u1) {
        if constexpr (S::NBUF == 1) __syncthreads();
        if constexpr (!EARLY) {
          ok = w.load(s_tiles);
          if (u + 2 < u1) w.find(kt.at(u + 2));
        }
        w.put(next);
        if (lane == 0) s_ok[flag ^ 1][w.wv] = ok;
        landed();
      }
      __syncthreads();
    }
  }
  w.l = half_sum(w.l);

  // the sums of the waves that share rows
  if constexpr (S::WK > 1) {
    constexpr int LD = S::LD;
    float* so = reinterpret_cast<float*>(s_tiles);
    float2* sm = reinterpret_cast<float2*>(so + 4 * 32 * LD);
    if (w.half == 0) sm[w.wv * 32 + w.col] = make_float2(w.m, w.l);
    __syncthreads();
    float top = NEG_INF, all = 0.0f;
#pragma unroll
    for (int k = 0; k < S::WK; ++k) top = fmaxf(top, sm[(w.wr * S::WK + k) * 32 + w.col].x);
    const float ref = top == NEG_INF ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < S::WK; ++k) {
      const float2 ml = sm[(w.wr * S::WK + k) * 32 + w.col];
      all += ml.y * __builtin_amdgcn_exp2f(ml.x - ref);
    }
    const float f = __builtin_amdgcn_exp2f(w.m - ref);
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<v4f*>(so + (w.wv * 32 + w.col) * LD + 32 * d + 2 * e + 4 * w.half) =
            v4f{w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]} * f;
    __syncthreads();
    w.m = top;
    w.l = all;
    // each wave of a row adds an equal share of the elements
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        if ((d * 4 + e / 4) % S::WK != w.wk) continue;
        v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < S::WK; ++k)
          x += *reinterpret_cast<const v4f*>(so + ((w.wr * S::WK + k) * 32 + w.col) * LD + 32 * d + 2 * e + 4 * w.half);
#pragma unroll
        for (int y = 0; y < 4; ++y) w.o[d][e + y] = x[y];
      }
  }
  if (mine >= rows) return;
  const float up = CT == BB_F16 ? F16_UP : 0.0f;
  if (kp.used == 1) {
    const bool none = w.m == NEG_INF && w.l == 0.0f;
    const float f = none ? 0.0f : 1.0f / w.l;
    const size_t at = (size_t)t * pq.out_stride + (size_t)head * kv.hd;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        if (S::WK > 1 && (d * 4 + e / 4) % S::WK != w.wk) continue;
        const int at0 = 32 * d + 2 * e + 4 * w.half;
        if (at0 < kv.hd)
          store_act(pq.out, at + at0, pq.dt, v4f{w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]} * f);
      }
    if (w.half == 0 && w.wk == 0 && pq.lse)
      pq.lse[(size_t)t * pq.n_heads + head] = none ? NEG_INF : (w.m + (__builtin_amdgcn_logf(w.l) - up)) * LN2;
  } else {
    const size_t slot = ((size_t)(g * pl.n_kv + kvh) * pl.parts + part) * S::BM + 32 * w.wr + w.col;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        if (S::WK > 1 && (d * 4 + e / 4) % S::WK != w.wk) continue;
        const int at0 = 32 * d + 2 * e + 4 * w.half;
        if (at0 < kv.hd)
          *reinterpret_cast<v4f*>(pl.sums + slot * kv.hd + at0) =
              v4f{w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]};
      }
    if (w.half == 0 && w.wk == 0) pl.ml[slot] = make_float2(w.m, w.l);
  }
}

// Adds the parts of a row (a wave), where there are several.
__global__ void __launch_bounds__(PP_THREADS) k_prompt_join(PromptQuery pq, int hd, int bm, PromptPlan pl, float up) {
  const int lane = threadIdx.x & 63, in = blockIdx.y * (PP_THREADS / 64) + (threadIdx.x >> 6);
  const int4 at = pl.places[blockIdx.x];
  const int used = at.x, r = at.y + in;
  if (used <= 1 || r >= at.z) return;
  const size_t first = (size_t)blockIdx.x * pl.parts * bm + in;
  float m = NEG_INF, l = 0.0f;
  for (int p = 0; p < used; ++p) m = fmaxf(m, pl.ml[first + (size_t)p * bm].x);
  const float ref = m == NEG_INF ? 0.0f : m;
  v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int p = 0; p < used; ++p) {
    const float2 ml = pl.ml[first + (size_t)p * bm];
    const float f = __builtin_amdgcn_exp2f(ml.x - ref);
    l += ml.y * f;
    if (4 * lane < hd) x += *reinterpret_cast<const v4f*>(pl.sums + (first + (size_t)p * bm) * hd + 4 * lane) * f;
  }
  const int t = at.w + r / pl.G, head = (int)(blockIdx.x % pl.n_kv) * pl.G + r % pl.G;
  const bool none = m == NEG_INF && l == 0.0f;
  if (4 * lane < hd)
    store_act(pq.out, (size_t)t * pq.out_stride + (size_t)head * hd + 4 * lane, pq.dt, x * (none ? 0.0f : 1.0f / l));
  if (lane == 0 && pq.lse)
    pq.lse[(size_t)t * pq.n_heads + head] = none ? NEG_INF : (m + (__builtin_amdgcn_logf(l) - up)) * LN2;
}

constexpr int PARTS_MAX = 64;

// The blocks of a launch, chosen from what the host knows: how many tokens and sequences there are.
struct PromptCut {
  bool few;  // tiles of 32 rows, the block's waves sharing its keys
  int bm, n_tiles, parts;
};
PromptCut prompt_cut(int n_cu, int cache, size_t n_tokens, size_t n_seqs, int G, int n_kv, int hd) {
  PromptCut c;
  const int cls = pa_class(hd);
  const size_t rows = n_tokens * (size_t)G, mean = (rows + n_seqs - 1) / n_seqs;
  c.few = mean <= 32 && !(cache == BB_F32 && cls == 256);
  c.bm = c.few ? 32 : 128;
  c.n_tiles = (int)std::min(rows / c.bm + n_seqs, rows);
  const size_t blocks = (size_t)c.n_tiles * n_kv;
  const size_t at_once = (size_t)n_cu * (cls == 256 || (cache == BB_F32 && cls == 128) ? 1 : 2);
  c.parts = (int)std::min<size_t>(PARTS_MAX, std::max<size_t>(1, at_once / blocks));
  return c;
}

size_t prompt_ws(const PromptCut& c, int n_kv, int hd) {
  if (c.parts == 1) return 0;
  const size_t tiles = (size_t)c.n_tiles * n_kv, slots = tiles * c.parts * c.bm;
  return slots * ((size_t)hd * 4 + sizeof(float2)) + tiles * sizeof(int4);
}

template <int CT, int NQ, int NP, int HDP, int WR, bool KV4>
hipError_t prompt_of(hipStream_t st, const PromptQuery& q, const PagedView& kv, const PagedSeqs& sq, PromptPlan pl) {
  typedef PpShape<CT, NQ, NP, HDP, WR, KV4> S;
  if constexpr (S::LDS > 159 * 1024) {
    return hipErrorInvalidValue;
  } else {
    // (no more parts than the table's width has of the least size)
    const size_t cap = ((size_t)sq.max_pages * kv.page_size + S::KT - 1) / S::KT;
    pl.least = std::max(1, 256 / S::KT);
    pl.parts = (int)std::min<size_t>(pl.parts, std::max<size_t>(1, cap / pl.least));
    const unsigned blocks = (unsigned)((size_t)pl.n_tiles * pl.n_kv * pl.parts);
    BB_LAUNCH((k_paged_prompt<CT, NQ, NP, HDP, WR, KV4>), dim3(blocks), dim3(PP_THREADS), 0, st, q, kv, sq, pl);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || pl.parts == 1) return e;
    BB_LAUNCH(k_prompt_join, dim3(pl.n_tiles * pl.n_kv, S::BM / (PP_THREADS / 64)), dim3(PP_THREADS), 0, st, q, kv.hd,
              S::BM, pl, CT == BB_F16 ? F16_UP : 0.0f);
    return hipGetLastError();
  }
}

template <int CT, int NQ, int NP, bool KV4>
hipError_t prompt_by(hipStream_t st, bool few, const PromptQuery& q, const PagedView& kv, const PagedSeqs& sq,
                     const PromptPlan& pl) {
  switch (pa_class(kv.hd)) {
    case 64: return few ? prompt_of<CT, NQ, NP, 64, 1, KV4>(st, q, kv, sq, pl) : prompt_of<CT, NQ, NP, 64, 4, KV4>(st, q, kv, sq, pl);
    case 128: return few ? prompt_of<CT, NQ, NP, 128, 1, KV4>(st, q, kv, sq, pl) : prompt_of<CT, NQ, NP, 128, 4, KV4>(st, q, kv, sq, pl);
    default: return few ? prompt_of<CT, NQ, NP, 256, 1, KV4>(st, q, kv, sq, pl) : prompt_of<CT, NQ, NP, 256, 4, KV4>(st, q, kv, sq, pl);
  }
}

}  // namespace

size_t paged_prompt_ws(int n_cu, int cache, size_t n_tokens, size_t n_seqs, int n_heads, int n_kv, int hd) {
  if (n_tokens == 0 || n_seqs == 0) return 0;
  return prompt_ws(prompt_cut(n_cu, cache, n_tokens, n_seqs, n_heads / n_kv, n_kv, hd), n_kv, hd);
}

// The types: a 16-bit cache takes 16-bit matrix instructions on its values as they are, a 4-bit one those of f16; the
// query rows are split into NQ parts that are all of them (f16 ones at a power of two that puts the row's
// largest in 2^13..2^14: f32 keeps 22 bits). Weights are rounded once to what the cache has (NP = 1: bf16 by 2^-9, f16 by
// 2^-12 at most) where out is rounded as far itself; an out with more bits has them in 2 or 3 parts.
hipError_t launch_paged_prompt(hipStream_t st, int n_cu, int cache, const PromptQuery& q, const PagedView& kv,
                               const PagedSeqs& sq) {
  const int G = q.n_heads / kv.n_kv;
  const PromptCut c = prompt_cut(n_cu, cache, q.n_tokens, sq.n_seqs, G, kv.n_kv, kv.hd);
  PromptPlan pl{G, c.n_tiles, kv.n_kv, c.parts, 1, nullptr, nullptr, nullptr};
  if (c.parts > 1) {
    const size_t tiles = (size_t)c.n_tiles * kv.n_kv, slots = tiles * c.parts * c.bm;
    pl.places = static_cast<int4*>(q.ws);
    pl.sums = reinterpret_cast<float*>(pl.places + tiles);
    pl.ml = reinterpret_cast<float2*>(pl.sums + slots * kv.hd);
  }
  switch (cache) {
    case BB_F32: return prompt_by<BB_F32, 1, 1, false>(st, c.few, q, kv, sq, pl);
    case BB_F16:
      return q.dt == BB_F32 ? prompt_by<BB_F16, 2, 2, false>(st, c.few, q, kv, sq, pl)
                            : prompt_by<BB_F16, 1, 1, false>(st, c.few, q, kv, sq, pl);
    case BB_BF16:
      return q.dt == BB_F32   ? prompt_by<BB_BF16, 3, 3, false>(st, c.few, q, kv, sq, pl)
             : q.dt == BB_F16 ? prompt_by<BB_BF16, 2, 2, false>(st, c.few, q, kv, sq, pl)
                              : prompt_by<BB_BF16, 1, 1, false>(st, c.few, q, kv, sq, pl);
    case BB_KV4:
      return q.dt == BB_F32 ? prompt_by<BB_F16, 2, 2, true>(st, c.few, q, kv, sq, pl)
                            : prompt_by<BB_F16, 1, 1, true>(st, c.few, q, kv, sq, pl);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bb
