// bb_paged_prompt.h — attention of several new tokens per sequence over a paged cache: prompts, chunks of
// them, drafts to verify (include/bebelm_moe.h states the operator). The reference has no counterpart. The kernels, which
// one source file for each type of cache instantiates (bb_prompt_*.hip); bb_paged_prompt.hip cuts a launch.
#ifndef BB_PAGED_PROMPT_H
#define BB_PAGED_PROMPT_H
#include <algorithm>
#include "bb_paged4.h"
#include "bb_paged_device.h"
#include "bb_prompt_plan.h"
#include "bb_prompt_turns.h"

namespace bb {

// The work of a launch: n_tiles (or fewer) tiles of rows, each for n_kv heads, its keys in up to `parts` parts of
// `least` tiles and more. The sums of parts, and for each tile and head (parts used, first row, rows and first token of
// its sequence), where there may be several.
struct PromptPlan {
  int G, n_tiles, n_kv, parts, least;
  bool runs;     // rows of a wave and a tile lie in one page (and fill theirs in LDS)
  float* sums;   // [tile][kv head][part][row][hd]
  float2* ml;    // [tile][kv head][part][row]: maximum (base 2), sum of weights
  int4* places;  // [tile][kv head]
};

namespace {

constexpr int PP_THREADS = 256;
// Weights go up to 2^SLACK, as f16 to 2^(SLACK + F16_UP) = 2^14, whose range then costs at most 2^-33 of the largest.
constexpr float SLACK = 6.0f, F16_UP = 8.0f;
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

// Where tiles come from: rows of the cache as they are; 4-bit ones, made f16; f32 ones, made sums of three bf16 parts each
// rounded from what the ones before leave (8 bits of it: all of 24 but 2^-25).
enum { SRC_SAME, SRC_KV4, SRC_PARTS };

// A block's shape. CT: the type that tiles have in LDS; WR waves along the rows (32 each), 4 / WR along the keys.
template <int CT, int NQ, int NP, int HDP, int WR, int SRC>
struct PpShape {
  static constexpr bool KV4 = SRC == SRC_KV4, PARTS = SRC == SRC_PARTS;
  static constexpr int SZ = CT == BB_F32 ? 4 : 2;
  static constexpr int NPL = PARTS ? 3 : 1;  // parts of an element, each a plane of the tile
  static constexpr int WK = 4 / WR, BM = 32 * WR;
  static constexpr int BN = WK > 1 || HDP * SZ >= 1024 || PARTS ? 32 : 64;  // keys of a wave's tile
  static constexpr int KT = WK * BN;                               // keys of the block's
  static constexpr int NT = BN / 32;
  // Rows in LDS: 16-byte pieces, of which row r has piece u at place u ^ k_swap(r) (keys) or u ^ v_swap(r) (values).
  // Keys are read a piece of 16 rows at once, 16-bit values 4 pieces of 4 rows, f32 values 8 pieces of
  // rows 4 apart: each time all banks.
  static constexpr int ROW = HDP * SZ, PPR = ROW / 16;
  __device__ static __forceinline__ int k_swap(int r) { return PPR == 8 ? r >> 1 & 7 : r & 15; }
  __device__ static __forceinline__ int v_swap(int r) {
    return SZ == 4 ? (r >> 2 & 1) << 3 : (PPR == 8 ? (r >> 1 & 1) << 2 : (r & 3) << 2) | (r >> 2 & 3);
  }
  static constexpr int PLANE = KT * ROW, BUF = 2 * NPL * PLANE;
  // (two of them: an iteration reads the keys of the next tile and the values of its own)
  static constexpr int LD = HDP + 4;                                        // a row of the waves' sums, in the same place
  static constexpr int SUMS = WK > 1 ? 4 * 32 * (LD * 4 + 8) : 4 * 32 * HDP * 4;
  static constexpr int LDS = 2 * BUF > SUMS ? 2 * BUF : SUMS;
  static constexpr int RPW = KT / 4;  // rows a wave brings
  // pieces of 16 bytes in LDS that a lane brings of keys (and of values); of a 4-bit cache, units of UE elements
  static constexpr int NPC = RPW * PPR / 64;
  // (of f32 parts, of 8)
  static constexpr int UE = PARTS ? 8 : RPW * HDP / 64 < 32 ? RPW * HDP / 64 : 32, UPR = HDP / UE, NU = RPW * UPR / 64;
  static constexpr int QW = CT == BB_F32 ? HDP / 2 : NQ * HDP / 4;  // registers of the query rows
  static constexpr int REGS = HDP / 2 + QW + 16 * NT + (CT == BB_F32 ? 0 : 8 * NP * NT) +
                              (KV4 ? 2 * NU * (UE / 8 + 1) : PARTS ? 16 * NU + 32 : 0);
  static constexpr int MOST = 160 * 1024 / (LDS + 64 * HDP + 64);  // blocks of a CU by their LDS
  static constexpr int WAVES = REGS <= 208 && MOST >= 2 ? 2 : 1;   // of a SIMD, and blocks of a CU
  // Shapes that are not used: tiles that do not fit, and one row of waves where its tiles leave one block a CU and query rows
  // of one part leave the matrix cores idle (16 x 5 tokens after 8192, heads of 128, bf16: 118 us, two rows 109; 64 x 5
  // after 2000 116 and 100; in three parts 125 and 174; one sequence 27.5 and 28.9).
  static constexpr bool NEVER = LDS > 159 * 1024 || (WR == 1 && WAVES == 1 && NQ == 1 && SZ == 2);
};

__device__ __attribute__((aligned(16))) uint32_t g_zeros[256];  // a row that is not there
// 16 bytes of every lane from its own address to lds + 16·lane.
__device__ __forceinline__ void to_lds(const char* from, char* lds) {
  typedef __attribute__((address_space(1))) const uint32_t* global_u32;
  typedef __attribute__((address_space(3))) uint32_t* lds_u32;
  __builtin_amdgcn_global_load_lds((global_u32)(from), (lds_u32)(lds), 16, 0, 0);
}
__device__ __forceinline__ uint32_t lds_at(const char* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)(p);
}
template <class T>
__device__ __forceinline__ T read_lds(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(uintptr_t)(at);
}
// (an address that is made again for every tile: dozens that follow from it would each take a register otherwise)
__device__ __forceinline__ uint32_t fresh(uint32_t a) {
  asm volatile("" : "+v"(a));
  return a;
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

// Two values as N bf16 parts, each rounded to the nearest.
template <int N>
__device__ __forceinline__ void round_parts(float a, float b, uint32_t (&w)[N]) {
  typedef __bf16 v2b __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const v2b r = {(__bf16)a, (__bf16)b};
    w[i] = __builtin_bit_cast(uint32_t, r);
    a = a - as_float(w[i] << 16);
    b = b - as_float(w[i] & 0xffff0000u);
  }
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


template <int CT, int NQ, int NP, int HDP, int WR, int SRC>
struct PpWave {
  typedef PpShape<CT, NQ, NP, HDP, WR, SRC> S;
  static constexpr int NT = S::NT, SZ = S::SZ, NPL = S::NPL;
  static constexpr bool KV4 = S::KV4, PARTS = S::PARTS;
  static constexpr int CZ = PARTS ? 4 : SZ;  // bytes of the cache's elements
  static constexpr bool F16 = CT == BB_F16;
  const PagedView& kv;
  const PromptQuery& pq;
  const int lane, col, half, wv, wr, wk;  // col: the wave's row that is the lane's
  const int* __restrict__ row;            // the sequence's page table
  size_t kv_off;
  int len, prefix;
  int i, lo;                  // the row's token's index, and what it sees first
  int i0, lo1;                // the index of the wave's first row, what its last sees first
  float c, slope;             // what scores are multiplied by; the bias of a step of distance (base 2)
  float m, l;
  v4u q[NQ][HDP / 16];
  v4f qf[CT == BB_F32 ? HDP / 8 : 1];
  v16f o[HDP / 32];
  struct Codes {
    uint32_t word[KV4 ? S::NU * S::UE / 8 : 1], head[KV4 ? S::NU : 1];
    v4u f32[PARTS ? 2 * S::NU : 1];
  };
  Codes ck, cv;
  v16f x[2][NT];              // scores of the tile at work (in multiples of `by`) and of the next, by turns
  float by;
  float top;                  // the largest
  bool runs;                  // a wave's rows of a tile lie in one page, a whole tile row each, within 2^31 bytes
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
      // (all of the row is asked for before any of it is used)
      typename RunOf<A, 8>::V in[HDP / 16][8 / RunOf<A, 8>::M];
#pragma unroll
      for (int j = 0; j < HDP / 16; ++j)
#pragma unroll
        for (int e = 0; e < 8; e += RunOf<A, 8>::M)
          in[j][e / RunOf<A, 8>::M] =
              *reinterpret_cast<const typename RunOf<A, 8>::V*>(p + min(16 * j + 8 * half, kv.hd - 8) + e);
      const auto element = [&](int j, int e) BB_INLINE { return (float)in[j][e / RunOf<A, 8>::M][e % RunOf<A, 8>::M]; };
      int up = 0;
      if constexpr (F16) {
        // the power of two that puts the row's largest in 2^13..2^14 (0 and what is not finite keep their scale)
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < HDP / 16; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(element(j, e)));
        top = half_max(top);
        up = top > 0.0f && top < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
        c = ldexpf(c, -up);
      }
#pragma unroll
      for (int j = 0; j < HDP / 16; ++j) {
        float x[8];
        const int d = 16 * j + 8 * half;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = element(j, e) * sign;
          x[e] = d < kv.hd ? F16 ? ldexpf(y, up) : y : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          uint32_t w[NQ];
          if constexpr (PARTS) round_parts(x[e], x[e + 1], w);
          else split2<CT, NQ>(x[e], x[e + 1], w);
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

  // Where the row found is in the pool (bytes; of 4 bits, to its (page, head)).
  struct Row {
    int64_t at;  // -1: not there
    int pos;     // 4 bits: its position in the page
    bool run;    // (the wave's) rows of one page, the first of which is there
  };
  __device__ __forceinline__ Row found() const {
    const bool there = (uint32_t)page < (uint32_t)kv.n_pages;
    const size_t at = (size_t)(uint32_t)page * kv.page_stride + (KV4 ? 0 : (size_t)(uint32_t)in * kv.pos_stride) + kv_off;
    return Row{there ? (int64_t)(KV4 ? at : at * CZ) : -1, in,
               runs && (uint32_t)__builtin_amdgcn_readfirstlane(page) < (uint32_t)kv.n_pages};
  }
  // Which of the wave's rows are there.
  static __device__ __forceinline__ uint32_t there(const Row& r) { return (uint32_t)__ballot(r.at >= 0) & (~0u >> (32 - S::RPW)); }

  // Asks for the wave's rows of a tile, keys or values: 4-bit ones into registers, others straight into the tile at
  // `lds`, 1024 bytes an instruction, each lane a piece. Rows of one page have one address and the lanes' distances from
  // it (those past the sequence's length are whatever is there: their scores are hidden, and look() finds values that are
  // not finite); otherwise the lanes exchange addresses, and rows that are not there are zeros.
  template <bool KEYS>
  __device__ __forceinline__ void load(const Row& w, char* lds) {
    const char* pool = static_cast<const char*>(KEYS ? kv.k : kv.v);
    if (w.run) {
      const uint64_t first = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(w.at >> 32)) << 32 |
                             (uint32_t)__builtin_amdgcn_readfirstlane((int)w.at);
      const char* base = pool + first;
      const uint32_t mine = fresh((uint32_t)lane) & 63;
      if constexpr (KV4) {
        Codes& c = KEYS ? ck : cv;
        const int in0 = __builtin_amdgcn_readfirstlane(w.pos);
        const char* heads = base + (size_t)(uint32_t)kv4_head_at(kv, in0, 0);
        const char* codes = base + (size_t)(uint32_t)(in0 * (kv.hd / 2));
#pragma unroll
        for (int p = 0; p < S::NU; ++p) {
          const uint32_t r = mine / S::UPR + p * (64 / S::UPR), u = mine % S::UPR;
          load_words<S::UE / 8>(codes + r * (HDP / 2) + u * (S::UE / 2), c.word + p * S::UE / 8);
          c.head[p] = *reinterpret_cast<const uint16_t*>(heads + 2 * (r * (HDP / 32) + u * S::UE / 32));
        }
      } else if constexpr (PARTS) {
        Codes& c = KEYS ? ck : cv;
        const uint32_t step = (uint32_t)kv.pos_stride * 4;
#pragma unroll
        for (int p = 0; p < S::NU; ++p) {
          const uint32_t r = mine / S::UPR + p * (64 / S::UPR), u = mine % S::UPR;
          c.f32[2 * p] = *reinterpret_cast<const v4u*>(base + (r * step + u * 32));
          c.f32[2 * p + 1] = *reinterpret_cast<const v4u*>(base + (r * step + u * 32 + 16));
        }
      } else {
        const uint32_t step = (uint32_t)kv.pos_stride * SZ, r0 = mine / S::PPR, u = mine % S::PPR;
#pragma unroll
        for (int p = 0; p < S::NPC; ++p) {
          const uint32_t r = r0 + p * (64 / S::PPR), rr = r + (wv * S::RPW & 15);
          const uint32_t at = (u ^ (uint32_t)(KEYS ? S::k_swap((int)rr) : S::v_swap((int)rr))) * 16;
          to_lds(base + (r * step + at), lds + wv * S::RPW * S::ROW + p * 1024);
        }
      }
      return;
    }
    const uint32_t own = fresh((uint32_t)lane) & 63;
    if constexpr (PARTS) {
      const uint32_t alo = (uint32_t)w.at, ahi = (uint32_t)(w.at >> 32);
      Codes& c = KEYS ? ck : cv;
#pragma unroll
      for (int p = 0; p < S::NU; ++p) {
        const int r = (int)(own / S::UPR) + p * (64 / S::UPR), u = own % S::UPR;
        const int64_t base = (int64_t)((uint64_t)(uint32_t)__shfl((int)ahi, r) << 32 | (uint32_t)__shfl((int)alo, r));
        c.f32[2 * p] = c.f32[2 * p + 1] = v4u{0, 0, 0, 0};
        if (base >= 0 && 8 * u < kv.hd) {
          c.f32[2 * p] = *reinterpret_cast<const v4u*>(pool + base + u * 32);
          c.f32[2 * p + 1] = *reinterpret_cast<const v4u*>(pool + base + u * 32 + 16);
        }
      }
    } else if constexpr (KV4) {
      const uint32_t alo = (uint32_t)w.at, ahi = (uint32_t)(w.at >> 32);
      Codes& c = KEYS ? ck : cv;
#pragma unroll
      for (int p = 0; p < S::NU; ++p) {
        const int r = (int)(own / S::UPR) + p * (64 / S::UPR), u = own % S::UPR, d = u * S::UE;
        const int64_t base = (int64_t)((uint64_t)(uint32_t)__shfl((int)ahi, r) << 32 | (uint32_t)__shfl((int)alo, r));
        const int rp = __shfl(w.pos, r);
        c.head[p] = 0;
#pragma unroll
        for (int i = 0; i < S::UE / 8; ++i) c.word[p * S::UE / 8 + i] = 0;
        if (base >= 0 && d < kv.hd) {
          load_words<S::UE / 8>(pool + base + (size_t)(uint32_t)(rp * (kv.hd / 2) + d / 2), c.word + p * S::UE / 8);
          c.head[p] = *reinterpret_cast<const uint16_t*>(pool + base + (size_t)(uint32_t)kv4_head_at(kv, rp, d / 32));
        }
      }
    } else {
      const uint64_t row = w.at >= 0 ? reinterpret_cast<uint64_t>(pool) + (uint64_t)w.at : reinterpret_cast<uint64_t>(g_zeros);
      const uint32_t alo = (uint32_t)row, ahi = (uint32_t)(row >> 32);
      // an instruction brings 64 / PPR rows (or a part of one); the addresses of several are asked for at once
      constexpr int AT_ONCE = S::NPC < 4 ? S::NPC : 4;
      const uint32_t r0 = own / S::PPR, u = own % S::PPR;
#pragma unroll
      for (int q = 0; q < S::NPC; q += AT_ONCE) {
        uint64_t a[AT_ONCE];
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          const int r = (int)(r0 + (q + p) * (64 / S::PPR)) * 4;
          a[p] = (uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(r, (int)ahi) << 32 |
                 (uint32_t)__builtin_amdgcn_ds_bpermute(r, (int)alo);
        }
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          const int r = (int)r0 + (q + p) * (64 / S::PPR) + wv * S::RPW;
          const uint32_t at = (u ^ (uint32_t)(KEYS ? S::k_swap(r) : S::v_swap(r))) * 16;
          a[p] += at;
          if (at >= (uint32_t)(kv.hd * SZ)) a[p] = reinterpret_cast<uint64_t>(g_zeros);  // (past a shorter head)
          to_lds(reinterpret_cast<const char*>(a[p]), lds + wv * S::RPW * S::ROW + (q + p) * 1024);
        }
      }
    }
  }

  // Puts 4-bit rows into a tile, as the f16 values they stand for, and f32 rows, as their parts.
  template <bool KEYS>
  __device__ __forceinline__ void put(char* lds) const {
    if constexpr (KV4) {
      const Codes& c = KEYS ? ck : cv;
      const Kv4Magic magic;
      const uint32_t own = fresh((uint32_t)lane) & 63;
#pragma unroll
      for (int p = 0; p < S::NU; ++p) {
        const int r = wv * S::RPW + (int)(own / S::UPR) + p * (64 / S::UPR), u = own % S::UPR;
        const Kv4Blocks block = Kv4Blocks::of(c.head[p]);
#pragma unroll
        for (int w = 0; w < S::UE / 8; ++w) {
          const int piece = u * (S::UE / 8) + w;
          *reinterpret_cast<v4u*>(lds + r * S::ROW + (piece ^ (KEYS ? S::k_swap(r) : S::v_swap(r))) * 16) =
              block.natural(c.word[p * S::UE / 8 + w], magic);
        }
      }
    }
    if constexpr (PARTS) {
      const Codes& c = KEYS ? ck : cv;
      const uint32_t own = fresh((uint32_t)lane) & 63;
#pragma unroll
      for (int p = 0; p < S::NU; ++p) {
        const int r = wv * S::RPW + (int)(own / S::UPR) + p * (64 / S::UPR), u = own % S::UPR;
        v4u part[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w[3];
          const v4u x = c.f32[2 * p + e / 2];
          round_parts(as_float(x[e % 2 * 2]), as_float(x[e % 2 * 2 + 1]), w);
#pragma unroll
          for (int i = 0; i < 3; ++i) part[i][e] = w[i];
        }
#pragma unroll
        for (int i = 0; i < 3; ++i)
          *reinterpret_cast<v4u*>(lds + i * S::PLANE + r * S::ROW + (u ^ (KEYS ? S::k_swap(r) : S::v_swap(r))) * 16) = part[i];
      }
    }
  }

  // Scores of a tile: register e of lane (row, half) is key 8(e / 4) + 4·half + e % 4 of 32. between(j) is done with the
  // products of the j-th of STEPS steps, whose keys have been asked for a step before.
  static constexpr int STEPS = HDP / 16, READS = CT == BB_F32 ? 2 : NPL;  // pieces of a step: of 16 elements, or of each part
  // (ALL: of all parts whose product counts, those of the first: 2^-23 of each other; otherwise of the first alone)
  template <bool ALL, class F>
  __device__ __forceinline__ void scores(uint32_t lk, v16f (&y)[NT], F&& between) const {
    const uint32_t at0 = fresh(lk + (wk * S::BN + col) * S::ROW + (half ^ S::k_swap(col)) * 16);
    const auto piece = [&](int j, int t, int l) BB_INLINE {
      return read_lds<v4u>((CT == BB_F32 ? at0 ^ 32 * (2 * j + l) : at0 ^ 32 * j) + 32 * t * S::ROW +
                           (CT == BB_F32 ? 0 : l * S::PLANE));
    };
    v4u a[2][NT][READS];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 16; ++e) y[t][e] = 0.0f;
#pragma unroll
      for (int l = 0; l < READS; ++l) a[0][t][l] = piece(0, t, l);
    }
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      if (j + 1 < STEPS)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int l = 0; l < READS; ++l) a[(j + 1) & 1][t][l] = piece(j + 1, t, l);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (CT == BB_F32) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(as_float(a[j & 1][t][e / 4][e % 4]), qf[2 * j + e / 4][e % 4], y[t],
                                                        0, 0, 0);
        } else {
#pragma unroll
          for (int i = NQ - 1; i >= 0; --i)
#pragma unroll
            for (int l = NPL - 1; l >= 0; --l)
              if (ALL ? l + i < 3 : l + i == 0) y[t] = mfma32<CT>(a[j & 1][t][l], q[i][j], y[t]);
        }
      }
      between(j);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Where the lane's values begin: at the keys of its registers 0 to 3 and, 16-bit types, 4 to 7.
  struct At {
    uint32_t a, b;
  };
  __device__ __forceinline__ At values_at(uint32_t lv) const {
    if constexpr (CT == BB_F32) {
      const int r = 4 * half;
      const uint32_t a = lv + (wk * S::BN + r) * S::ROW + (col / 4 ^ S::v_swap(r)) * 16 + col % 4 * 4;
      return At{fresh(a), 0};
    } else {
      const int r = 4 * half + (lane & 15) / 4, piece = (lane & 16) / 8 + (lane & 2) / 2;
      const uint32_t row = lv + (wk * S::BN + r) * S::ROW + (lane & 1) * 8;
      return At{fresh(row + (piece ^ S::v_swap(r)) * 16), fresh(row + 8 * S::ROW + (piece ^ S::v_swap(r + 8)) * 16)};
    }
  }
  // Elements 32·dt + lane % 32 of the values at the keys whose weights are registers 8s..8s+7 of a tile (16-bit types).
  __device__ __forceinline__ v4u values(At at, int t, int s, int dt, int plane = 0) const {
    typedef __attribute__((address_space(3))) v4s* lds_v4s;
    const int more = (32 * t + 16 * s) * S::ROW + plane * S::PLANE;
    const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)((at.a ^ 64 * dt) + more));
    const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)((at.b ^ 64 * dt) + more));
    const v2u x = __builtin_bit_cast(v2u, a), y = __builtin_bit_cast(v2u, b);
    return v4u{x[0], x[1], y[0], y[1]};
  }
  // (the same of an f32 cache: at the key of register e)
  __device__ __forceinline__ float value(At at, int t, int e, int dt) const {
    return read_lds<float>((at.a ^ 128 * dt) + (32 * t + 8 * (e / 4) + e % 4) * S::ROW);
  }

  // Which of 32 keys from j0 on the row sees, of those in `ok`: the bits of the lane's registers e at 8(e / 4) + e % 4.
  __device__ __forceinline__ uint32_t seen(int j0, uint32_t ok) const {
    const auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; };  // keys 0..n-1
    return ((below(i + 1 - j0) & ~below(lo - j0)) | below(prefix - j0)) & ok;
  }

  // The scores of a tile of keys, into set I.
  template <int I, class F>
  __device__ __forceinline__ void score(uint32_t lk, F&& between) {
    v16f(&y)[NT] = x[I];
    scores<true>(lk, y, between);
    if constexpr (NQ > 1) {
      // a part of 0 meets an infinite key as NaN: such scores are taken from the first parts alone
      bool odd = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) odd |= y[t][e] != y[t][e];
      if (__any(odd)) {
        v16f z[NT];
        scores<false>(lk, z, [](int) {});
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) y[t][e] = y[t][e] != y[t][e] ? z[t][e] : y[t][e];
      }
    }
  }

  // Whether all rows of the wave see all keys from j0 on, `ok` being those that are there.
  __device__ __forceinline__ bool whole(int j0, uint32_t ok0, uint32_t ok1) const {
    return ok0 == ~0u && (NT == 1 || ok1 == ~0u) && ((j0 + S::BN - 1 <= i0 && j0 >= lo1) || j0 + S::BN <= prefix);
  }

  // cap·tanh as cap - 2cap / (exp(2y) + 1): off by at most 2^-21 of the cap (the quotient's roundings and the
  // sum's), however small the score. Up to a cap of QUICK_CAP that is 2^-15 of a weight, an eighth of the half step by which f16
  // rounds it, and of the log sum; larger ones take capped(), which is off by a few steps of the score itself. It has half the
  // instructions of that (6001 tokens, 16 heads of 256, f16: the whole call 297 us with that and 254 with this).
  static constexpr bool QUICK = CT != BB_F32 && NP == 1;
  static constexpr float QUICK_CAP = 64.0f;
  // (y·twice: two capless scores by the cap, as an exponent of 2)
  __device__ __forceinline__ float quick_cap(float y, float twice) const {
    const float e = __builtin_amdgcn_exp2f(y * twice);
    return fmaf(-2.0f * pq.cap.top, __builtin_amdgcn_rcpf(e + 1.0f), pq.cap.top);
  }
  // The scores capped, with their bias, hidden where the rows do not see the keys from j0 on, and the largest.
  template <int I>
  __device__ __forceinline__ void shape(int j0, uint32_t ok0, uint32_t ok1) {
    v16f(&y)[NT] = x[I];
    by = c;
    if (pq.cap.top > 0.0f) {
      by = 1.0f;
      if (QUICK && pq.cap.top <= QUICK_CAP * LOG2E) {
        // (finite: 0 times it is 0)
        const float twice = fminf(c * (pq.cap.inv * (2.0f * LOG2E)), 3.0e38f);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) y[t][e] = quick_cap(y[t][e], twice);
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) y[t][e] = capped(y[t][e] * c, pq.cap);
      }
    }
    if (pq.slopes) {
      const float away = (float)(i - j0 - 4 * half);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          y[t][e] = fmaf(-slope, fabsf(away - (float)(32 * t + 8 * (e / 4) + e % 4)), y[t][e] * by);
      by = 1.0f;
    }
    if (!whole(j0, ok0, ok1)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t see = seen(j0 + 32 * t, t ? ok1 : ok0) >> 4 * half;
#pragma unroll
        for (int e = 0; e < 16; ++e) y[t][e] = see >> (8 * (e / 4) + e % 4) & 1 ? y[t][e] : NEG_INF;
      }
    }
    float mx = NEG_INF;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, y[t][e]);
    top = half_max(mx) * by;
  }

  // The running maximum stays until a score is SLACK past it: the sums are as exact, and seldom multiplied.
  // (by the difference: m + SLACK may be rounded to a maximum two steps of 4 or one of 8 away, whose weight f16 does not hold)
  __device__ __forceinline__ bool past() const { return __any(top - m > SLACK); }
  __device__ __forceinline__ void raise() {
    const float mx = top - m > SLACK ? top : m;
    const float f = __builtin_amdgcn_exp2f(m - (mx == NEG_INF ? 0.0f : mx));
    m = mx;
    l *= f;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] *= f;
  }

  // A weight is 2^(x·by - m) by one multiply-add: what -m + F16_UP is rounded by, and m was as a product, goes into the
  // exponent, of all of a row's weights alike while m stays. From FAR on, where that may be 2^-7, a row's scores are made
  // differences from m beforehand, of the product that m was taken of, and its m is 0 while they are weighed. (Each row by its own
  // m: one that did so for a neighbour's sake would have weights of two kinds.)
  static constexpr float FAR = 65536.0f;
  __device__ __forceinline__ bool far_row() const { return fabsf(m) >= FAR && m != NEG_INF; }
  __device__ __forceinline__ bool far() const { return __any(far_row()); }
  __device__ __forceinline__ float near() {
    const float kept = m;
    if (far_row()) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[0][t][e] = x[0][t][e] * by - m;
      by = 1.0f;
      m = 0.0f;
    }
    return kept;
  }

  // The weights of the tile, in 16 bits: register 2e of w[t][s][part] those of registers 8s + 2e and 8s + 2e + 1.
  struct Weights {
    v4u w[CT == BB_F32 ? 1 : NT][2][NP];
    v16f f[CT == BB_F32 ? NT : 1];
  };
  // Those of pairs of registers lo..hi-1 (8 of each 32 keys).
  template <int I>
  __device__ __forceinline__ void weigh(Weights& p, int lo, int hi) {
    const float less = (F16 ? F16_UP : 0.0f) - (m == NEG_INF ? 0.0f : m);
#pragma unroll
    for (int i = lo; i < hi; ++i) {
      const int t = i / 8, e = i % 8 * 2;
      const float a = __builtin_amdgcn_exp2f(fmaf(x[I][t][e], by, less));
      const float b = __builtin_amdgcn_exp2f(fmaf(x[I][t][e + 1], by, less));
      l += a;
      l += b;
      asm("" : "+v"(l));  // (here, not when all weights are there)
      if constexpr (CT == BB_F32) {
        p.f[t][e] = a;
        p.f[t][e + 1] = b;
      } else {
        uint32_t w[NP];
        split2<CT, NP>(a, b, w);
#pragma unroll
        for (int k = 0; k < NP; ++k) p.w[t][e / 8][k][e % 8 / 2] = w[k];
      }
    }
  }

  // Whether the rows that the wave brings have values that are not finite (of parts, the first is it).
  __device__ __forceinline__ bool values_odd(uint32_t lv) const {
    constexpr uint32_t EXP = CT == BB_BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = CT == BB_BF16 ? 0x00800080u : 0x04000400u;
    uint32_t odd = 0;
#pragma unroll 4
    for (int i = lane; i < S::RPW * S::PPR; i += 64) {
      const v4u a = read_lds<v4u>(lv + (wv * S::RPW * S::PPR + i) * 16);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        odd |= CT == BB_F32 ? (a[w] & 0x7f800000u) + 0x00800000u : (a[w] & EXP) + ONE;  // (carries into the sign's place)
    }
    return (odd & 0x80008000u) != 0;
  }

  // The values times their weights.
  __device__ __forceinline__ void add(uint32_t lv, const Weights& p) {
    const At at = values_at(lv);
    constexpr int ND = HDP / 32;
    if constexpr (CT == BB_F32) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int d = 0; d < ND; ++d)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(value(at, t, e, d), p.f[t][e], o[d], 0, 0, 0);
    } else {
      // (four of them at a time, asked for four ahead)
      constexpr int DC = ND < 4 ? ND : 4, N = 2 * NT * ND / DC;
      v4u a[2][DC][NPL];
      const auto ask = [&](int i) BB_INLINE {
        const int g = i / (ND / DC);
#pragma unroll
        for (int d = 0; d < DC; ++d)
#pragma unroll
          for (int l = 0; l < NPL; ++l) a[i & 1][d][l] = values(at, g / 2, g % 2, i % (ND / DC) * DC + d, l);
      };
      ask(0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + 1 < N) ask(i + 1);
        const int g = i / (ND / DC);
#pragma unroll
        for (int d = 0; d < DC; ++d)
#pragma unroll
          for (int k = NP - 1; k >= 0; --k)
#pragma unroll
            for (int l = NPL - 1; l >= 0; --l)
              if (l + k < 3)
                o[i % (ND / DC) * DC + d] = mfma32<CT>(a[i & 1][d][l], p.w[g / 2][g % 2][k], o[i % (ND / DC) * DC + d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // Which sums a value that is not finite belongs to, among those a row sees of a tile: bit e of the lane's bad[d], by
  // products as those of the sums, of ones.
  __device__ __forceinline__ void mark(uint32_t* bad, uint32_t lv, int j0, uint32_t ok0, uint32_t ok1) const {
    const At at = values_at(lv);
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d) {
      v16f n;
#pragma unroll
      for (int e = 0; e < 16; ++e) n[e] = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t see = seen(j0 + 32 * t, t ? ok1 : ok0) >> 4 * half;
        const auto bit = [&](int e) BB_INLINE { return see >> (8 * (e / 4) + e % 4) & 1; };
        if constexpr (CT == BB_F32) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float a = fabsf(value(at, t, e, d)) < __builtin_inff() ? 0.0f : 1.0f;
            n = __builtin_amdgcn_mfma_f32_32x32x2f32(a, (float)bit(e), n, 0, 0, 0);
          }
        } else {
          constexpr uint32_t ONE = CT == BB_BF16 ? 0x3f80u : 0x3c00u;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            v4u a = values(at, t, s, d), p;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              a[w] = odd_halves<CT>(a[w]);
              p[w] = (bit(8 * s + 2 * w) ? ONE : 0u) | (bit(8 * s + 2 * w + 1) ? ONE << 16 : 0u);
            }
            n = mfma32<CT>(a, p, n);
          }
        }
      }
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) bits |= (n[e] > 0.0f ? 1u : 0u) << e;
      bad[d * PP_THREADS] = bits;
    }
  }
  __device__ __forceinline__ void spoil(const uint32_t* bad) {
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = bad[d * PP_THREADS] >> e & 1 ? __builtin_nanf("") : o[d][e];
  }
  // The rows that the wave brings without values that are not finite.
  __device__ __forceinline__ void clean(char* lv) const {
    for (int i = lane; i < NPL * S::RPW * S::PPR; i += 64) {
      const int l = i / (S::RPW * S::PPR), in = i % (S::RPW * S::PPR);
      v4u* p = reinterpret_cast<v4u*>(lv + l * S::PLANE + (wv * S::RPW * S::PPR + in) * 16);
      v4u a = *p;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        a[w] = CT == BB_F32 ? (a[w] & 0x7f800000u) == 0x7f800000u ? 0u : a[w] : fine_halves(a[w], odd_halves<CT>(a[w]));
      *p = a;
    }
  }
};

// A block's steps, a wave's share of them, for PromptTurns.
template <int CT, int NQ, int NP, int HDP, int WR, int SRC>
struct PpBlock {
  typedef PpShape<CT, NQ, NP, HDP, WR, SRC> S;
  typedef PpWave<CT, NQ, NP, HDP, WR, SRC> Wave;
  Wave& w;
  const KeyTiles& kt;
  char* const tiles;
  uint32_t (&s_ok)[2][4];
  uint32_t (&s_odd)[2][4];
  uint32_t (&s_marks)[2][HDP / 32][PP_THREADS];
  const int u0, b0, b1;  // b0, b1: the least that all rows of the block see is up to b0, from b1 on
  typename Wave::Row krow, vrow;
  uint32_t ok0, ok1;

  __device__ BB_INLINE char* keys_of(int u) const { return tiles + (u & 1) * S::BUF; }
  __device__ BB_INLINE char* vals_of(int u) const { return tiles + (u & 1) * S::BUF + S::NPL * S::PLANE; }
  __device__ BB_INLINE int first_key(int u) const { return kt.at(u0 + u) * S::KT + w.wk * S::BN; }
  __device__ BB_INLINE void flags(int u) {
    const uint32_t* ok = s_ok[u & 1];
    ok1 = ~0u;
    if constexpr (S::RPW == 32) {
      ok0 = ok[w.wk];
    } else if constexpr (S::WK == 1 && S::RPW == 16) {
      ok0 = ok[0] | ok[1] << 16;
      ok1 = ok[2] | ok[3] << 16;
    } else if constexpr (S::WK == 2) {
      ok0 = ok[2 * w.wk] | ok[2 * w.wk + 1] << 16;
    } else {
      ok0 = ok[0] | ok[1] << 8 | ok[2] << 16 | ok[3] << 24;
    }
    ok0 = __builtin_amdgcn_readfirstlane(ok0);
    ok1 = __builtin_amdgcn_readfirstlane(ok1);
  }

  __device__ BB_INLINE void find(int u) { w.find(kt.at(u0 + u)); }
  __device__ BB_INLINE void keys(int u) {
    krow = w.found();
    const uint32_t ok = Wave::there(krow);
    if (w.lane == 0) s_ok[u & 1][w.wv] = ok;
    w.template load<true>(krow, keys_of(u));
  }
  __device__ BB_INLINE void pass() { vrow = krow; }
  __device__ BB_INLINE void values(int u) { w.template load<false>(vrow, vals_of(u)); }
  __device__ BB_INLINE void put_keys(int u) { w.template put<true>(keys_of(u)); }
  __device__ BB_INLINE void put_values(int u) { w.template put<false>(vals_of(u)); }
  __device__ BB_INLINE void landed() { bb::landed(); }
  __device__ BB_INLINE void barrier() { __syncthreads(); }
  template <int I>
  __device__ BB_INLINE void score(int u, Set<I>) {
    w.template score<I>(lds_at(keys_of(u)), [](int) {});
  }
  template <int I>
  __device__ BB_INLINE void see(int u, Set<I>) {
    flags(u);
    w.template shape<I>(first_key(u), ok0, ok1);
  }
  template <int I, class F>
  __device__ BB_INLINE void products(int u, Set<I>, F&& ask) {
    typename Wave::Weights p;
    __builtin_amdgcn_sched_barrier(0);
    // (behind the last tile, scores of whatever is there, for nothing)
    w.template score<1 - I>(lds_at(keys_of(u + 1)), [&](int j) BB_INLINE {
      constexpr int PAIRS = 8 * S::NT;
      ask(j);
      w.template weigh<I>(p, j * PAIRS / Wave::STEPS, (j + 1) * PAIRS / Wave::STEPS);
    });
    w.add(lds_at(vals_of(u)), p);
  }
  __device__ BB_INLINE bool shared(int u) const {
    const int j0 = kt.at(u0 + u) * S::KT;
    return (j0 + S::KT - 1 <= b0 && j0 >= b1) || j0 + S::KT <= w.prefix;
  }
  __device__ BB_INLINE bool odd(int u) const { return __ballot(w.values_odd(lds_at(vals_of(u)))) != 0; }
  __device__ BB_INLINE void tell(int at, bool mine) {
    if (w.lane == 0) s_odd[at][w.wv] = mine;
  }
  __device__ BB_INLINE bool told(int at) const { return (s_odd[at][0] | s_odd[at][1] | s_odd[at][2] | s_odd[at][3]) != 0; }
  __device__ BB_INLINE uint32_t* marks(int u) const { return &s_marks[u & 1][0][threadIdx.x]; }
  __device__ BB_INLINE void mark(int u) { w.mark(marks(u), lds_at(vals_of(u)), first_key(u), ok0, ok1); }
  __device__ BB_INLINE void clean(int u) { w.clean(vals_of(u)); }
  __device__ BB_INLINE void spoil(int u) { w.spoil(marks(u)); }
  __device__ BB_INLINE bool past() const { return w.past(); }
  __device__ BB_INLINE void raise() { w.raise(); }
  __device__ BB_INLINE bool far() const { return w.far(); }
  // (m in the place of the next tile's marks, which are made after back())
  __device__ BB_INLINE void near(int u) { *marks(u + 1) = __float_as_uint(w.near()); }
  __device__ BB_INLINE void back(int u) { w.m = as_float(*marks(u + 1)); }
  __device__ BB_INLINE void last() {
#pragma unroll
    for (int t = 0; t < S::NT; ++t) w.x[0][t] = w.x[1][t];
  }
};

// out[t][h] = sum_j softmax_j(x[t][h][j])·v[j], a tile of rows (the G query heads of adjacent tokens, which share a kv head) in
// one pass over the keys that any of them sees, with the running maximum and sum of the softmax.
//
// The scores are made transposed, Sᵀ = K·Qᵀ, by 32x32 matrix instructions: a lane then has scores of one row, 4 adjacent keys
// at a time, which as weights are the second operand of Oᵀ = Vᵀ·Pᵀ just where they are; Vᵀ comes from LDS by reads that
// transpose. Nothing moves between lanes but the two halves of a row's maximum. Query rows and sums stay in
// registers. Keys and values go to LDS without passing registers, in an order of 16-byte pieces that leaves no bank
// conflict (4 bits and f32 parts pass them, to be made 16-bit). Tiles that all rows see skip masks; those that
// have something to be hidden get them as bits.
//
// What bounds it: matrix instructions and, nearly added to them, the vector ones (a weight is a multiply-add, an
// exponential, a sum and half a conversion). 16384 tokens from the first, 32 heads on 8 of 128, bf16: 2.23 to 2.49 ms by the card, 880 to
// 985 TFLOP/s, where large products reach 1120 (keys by way of registers 8.3 ms; straight to LDS, with a maximum that
// seldom moves, 3.3; a tile's weights made while the next one's scores are, 2.8; without spills 2.7; a page's
// rows by one address and their loads behind the first products 2.3). 5003 tokens of 7 ragged prompts, 13 tiles a block: 111 to 119 us,
// 590 to 630 TFLOP/s; blocks begin and end (6 us) two or three times a CU, and the last are alone. Heads of 256 fill the
// registers of a SIMD with one wave, whose vector, matrix and LDS work then follow each other: 6001 tokens with a cap and a
// window of 1024, f16, 191 to 203 us, 410 to 440 TFLOP/s. From 4 bits (2048 tokens after 8192, heads of 128) 374 to 408 us, 690 to
// 755 TFLOP/s: 150 vector instructions a tile and wave make f16 of the codes. 5 tokens of each of 16 sequences after 8192: 108 us,
// 5.0 TB/s of cache.
template <int CT, int NQ, int NP, int HDP, int WR, int SRC>
__global__ void __launch_bounds__(PP_THREADS, (PpShape<CT, NQ, NP, HDP, WR, SRC>::WAVES))
    k_paged_prompt(PromptQuery pq, PagedView kv, PagedSeqs sq, PromptPlan pl) {
  typedef PpShape<CT, NQ, NP, HDP, WR, SRC> S;
  __shared__ __align__(1024) char s_tiles[S::LDS];
  __shared__ uint32_t s_ok[2][4];
  __shared__ uint32_t s_odd[2][4];
  __shared__ uint32_t s_marks[2][HDP / 32][PP_THREADS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kvh = blockIdx.x % pl.n_kv, rest = blockIdx.x / pl.n_kv;
  const int part = rest % pl.parts, g = rest / pl.parts;

  // the sequence whose tile this is (every wave by itself); of a sequence the tiles that see most come first
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
      it = before + __builtin_amdgcn_readlane(incl, at) - 1 - g;
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

  typedef PpWave<CT, NQ, NP, HDP, WR, SRC> Wave;
  Wave w(kv, pq, tid);
  const int raw = sq.lens[s], end = pq.seq_start ? pq.seq_start[s + 1] : s + 1;
  w.len = min(max(raw, 0), sq.max_pages * kv.page_size);
  w.prefix = pq.prefix ? min(max(pq.prefix[s], 0), w.len) : 0;
  w.runs = pl.runs;
  w.row = sq.table + (size_t)s * sq.table_stride;
  w.kv_off = (size_t)kvh * kv.head_stride;
  const int rows = n * pl.G, r0 = it * S::BM;
  const auto index_of = [&](int r) { return token_index(w.len, end, a + r / pl.G); };
  const KeyTiles kt =
      key_tiles(index_of(r0), index_of(min(r0 + S::BM, rows) - 1), w.len, w.prefix, pq.window, S::KT);
  const KeyParts kp = key_parts(kt.n, pl.parts, pl.least);
  if (part >= kp.used) return;
  if (part == 0 && tid == 0 && pl.parts > 1) pl.places[g * pl.n_kv + kvh] = make_int4(kp.used, r0, rows, a);
  const int u0 = part * kp.per, u1 = min(kt.n, u0 + kp.per);

  const int mine = r0 + 32 * w.wr + w.col, r = min(mine, rows - 1);
  const int t = a + r / pl.G, head = kvh * pl.G + r % pl.G;
  w.i = token_index(w.len, end, t);
  w.lo = first_seen(w.i, pq.window);
  w.i0 = __builtin_amdgcn_readlane(w.i, 0);
  w.lo1 = __builtin_amdgcn_readlane(w.lo, 31);
  w.slope = pq.slopes ? pq.slopes[head] * LOG2E : 0.0f;
  w.c = fabsf(pq.scale) * LOG2E;
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
    w.c = fmaxf(w.c, 1e-45f);  // (0 times an infinite score would be NaN)
  }

  // Tiles u0..u1-1 (bb_prompt_turns.h).
  if (u0 < u1) {
    const int last = min(r0 + S::BM, rows) - 1;
    typedef PpBlock<CT, NQ, NP, HDP, WR, SRC> Block;
    Block b{w, kt, s_tiles, s_ok, s_odd, s_marks, u0, index_of(r0), first_seen(index_of(last), pq.window), {}, {}, 0, 0};
    PromptTurns<Block>(b, u1 - u0).run();
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
  const float up = CT == BB_F16 ? F16_UP : 0.0f;
  const bool all = kp.used == 1, none = w.m == NEG_INF && w.l == 0.0f;
  const float f = !all ? 1.0f : none ? 0.0f : 1.0f / w.l;
  const size_t slot = all ? 0 : ((size_t)(g * pl.n_kv + kvh) * pl.parts + part) * S::BM + 32 * w.wr + w.col;
  const size_t to = all ? (size_t)t * pq.out_stride + (size_t)head * kv.hd : slot * kv.hd;
  const auto store = [&](size_t at, const v4f& x) BB_INLINE {
    if (all) store_act(pq.out, at, pq.dt, x);
    else *reinterpret_cast<v4f*>(pl.sums + at) = x;
  };
  if (mine < rows && w.half == 0 && w.wk == 0) {
    if (!all) pl.ml[slot] = make_float2(w.m, w.l);
    else if (pq.lse)
      pq.lse[(size_t)t * pq.n_heads + head] = none ? NEG_INF : (w.m + (__builtin_amdgcn_logf(w.l) - up)) * LN2;
  }
  if constexpr (S::WK > 1) {
    if (mine >= rows) return;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        if ((d * 4 + e / 4) % S::WK != w.wk) continue;
        const int at0 = 32 * d + 2 * e + 4 * w.half;
        if (at0 < kv.hd) store(to + at0, v4f{w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]} * f);
      }
  } else {
    // by way of LDS, a wave its own rows, so that a row's stores are adjacent (straight from the registers, where a lane has 4
    // elements of every 32 of its own row, they cost 6 us a block). Piece p of row r lies at p ^ r % 16.
    constexpr int P4 = HDP / 4;
    v4f* rows_at = reinterpret_cast<v4f*>(s_tiles) + w.wv * 32 * P4;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        rows_at[w.col * P4 + ((8 * d + e / 2 + w.half) ^ (w.col & 15))] =
            v4f{w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]} * f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int left = rows - (r0 + 32 * w.wr);  // rows of the wave that are there
    const uint32_t lo = (uint32_t)to, hi = (uint32_t)(to >> 32);
#pragma unroll 4
    for (int i = lane; i < 32 * P4; i += 64) {
      const int row = i / P4, piece = i % P4;
      const size_t at = (size_t)(uint32_t)__shfl((int)hi, row) << 32 | (uint32_t)__shfl((int)lo, row);
      if (row < left && 4 * piece < kv.hd) store(at + 4 * piece, rows_at[row * P4 + (piece ^ (row & 15))]);
    }
  }
}


// f(a block's shape) by the types of the cache and of q and out, the head size and the waves along the rows (4, 2 or 1).
//
// A 16-bit cache takes 16-bit matrix instructions on its values as they are, a 4-bit one those of f16; the query rows are split
// into NQ parts that are all of them (f16 ones at a power of two that puts the row's largest in 2^13..2^14: f32
// keeps 22 bits). Weights are rounded once to what the cache has (NP = 1: bf16 by 2^-8, f16 by 2^-11 at most) where out
// is rounded as far itself; an out with more bits has them in 2 or 3 parts. An f32 cache takes f32 instructions, or for
// tiles of 128 rows and heads of up to 128 (more parts do not fit LDS) six times 16-bit ones (of the products of three
// parts with three, those that count), of a sixteenth of the time each: 512 tokens after 1536, heads of 64, 67 us instead of
// 104, 17 tokens 8.3 instead of 13.4. Few rows leave such a tile mostly empty: 8 x 5 tokens after 8192, heads of 64, 118
// us, with f32 instructions and the keys shared out 68.
template <int CT, int NQ, int NP, int SRC, class F>
auto by_size(int cls, int wr, F& f) {
  const auto of = [&](auto hdp) {
    constexpr int H = decltype(hdp)::value;
    return wr == 4   ? f(PpShape<CT, NQ, NP, H, 4, SRC>())
           : wr == 2 ? f(PpShape<CT, NQ, NP, H, 2, SRC>())
                     : f(PpShape<CT, NQ, NP, H, 1, SRC>());
  };
  return cls == 64    ? of(std::integral_constant<int, 64>())
         : cls == 128 ? of(std::integral_constant<int, 128>())
                      : of(std::integral_constant<int, 256>());
}
template <class F>
auto shape_f32(int dt, int cls, int wr, F&& f) {
  if (wr == 4 && cls < 256) {
    if (dt == BB_F32) return cls == 64 ? f(PpShape<BB_BF16, 3, 3, 64, 4, SRC_PARTS>()) : f(PpShape<BB_BF16, 3, 3, 128, 4, SRC_PARTS>());
    return cls == 64 ? f(PpShape<BB_BF16, 2, 3, 64, 4, SRC_PARTS>()) : f(PpShape<BB_BF16, 2, 3, 128, 4, SRC_PARTS>());
  }
  return by_size<BB_F32, 1, 1, SRC_SAME>(cls, wr, f);
}
template <class F>
auto shape_f16(int dt, int cls, int wr, F&& f) {
  return dt == BB_F32 ? by_size<BB_F16, 2, 2, SRC_SAME>(cls, wr, f) : by_size<BB_F16, 1, 1, SRC_SAME>(cls, wr, f);
}
template <class F>
auto shape_kv4(int dt, int cls, int wr, F&& f) {
  return dt == BB_F32 ? by_size<BB_F16, 2, 2, SRC_KV4>(cls, wr, f) : by_size<BB_F16, 1, 1, SRC_KV4>(cls, wr, f);
}
template <class F>
auto shape_bf16(int dt, int cls, int wr, F&& f) {
  return dt == BB_F32   ? by_size<BB_BF16, 3, 3, SRC_SAME>(cls, wr, f)
         : dt == BB_F16 ? by_size<BB_BF16, 2, 2, SRC_SAME>(cls, wr, f)
                        : by_size<BB_BF16, 1, 1, SRC_SAME>(cls, wr, f);
}

template <int CT, int NQ, int NP, int HDP, int WR, int SRC>
hipError_t prompt_of(PpShape<CT, NQ, NP, HDP, WR, SRC>, hipStream_t st, const PromptQuery& q, const PagedView& kv,
                     const PagedSeqs& sq, PromptPlan& pl) {
  typedef PpShape<CT, NQ, NP, HDP, WR, SRC> S;
  if constexpr (S::NEVER) {
    return hipErrorInvalidValue;  // (prompt_cut chooses none of these)
  } else {
    // (no more parts than the table's width has of the least size)
    const size_t cap = ((size_t)sq.max_pages * kv.page_size + S::KT - 1) / S::KT;
    pl.least = std::max(1, 256 / S::KT);
    pl.runs = kv.page_size % S::RPW == 0 && kv.hd == HDP && (size_t)S::RPW * kv.pos_stride * 4 < ((size_t)1 << 31);
    pl.parts = (int)std::min<size_t>(pl.parts, std::max<size_t>(1, cap / pl.least));
    const unsigned blocks = (unsigned)((size_t)pl.n_tiles * pl.n_kv * pl.parts);
    BB_LAUNCH((k_paged_prompt<CT, NQ, NP, HDP, WR, SRC>), dim3(blocks), dim3(PP_THREADS), 0, st, q, kv, sq, pl);
    return hipGetLastError();
  }
}

}  // namespace

// The main launch for a cache of one type (pl.least, runs and parts are settled).
hipError_t launch_prompt_f32(hipStream_t st, int wr, const PromptQuery& q, const PagedView& kv, const PagedSeqs& sq, PromptPlan& pl);
hipError_t launch_prompt_f16(hipStream_t st, int wr, const PromptQuery& q, const PagedView& kv, const PagedSeqs& sq, PromptPlan& pl);
hipError_t launch_prompt_bf16(hipStream_t st, int wr, const PromptQuery& q, const PagedView& kv, const PagedSeqs& sq, PromptPlan& pl);
hipError_t launch_prompt_kv4(hipStream_t st, int wr, const PromptQuery& q, const PagedView& kv, const PagedSeqs& sq, PromptPlan& pl);

}  // namespace bb
#endif
