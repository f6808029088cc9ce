// bb_paged4.h — the blocks of a 4-bit paged cache: 32 elements of a head row, 16 bytes of codes (element 2i in the low
// half of byte i) and a 16-bit head with the step d (bits 6 to 14: an f16 number of 5 significant bits) and the
// offset z (bits 0 to 5, bit 15 for -64). An element stands for d·(code + z): with code + z in -47..63 that is 6 bits
// times 5, exact in f16, so that the matrix cores' 16-bit instructions take it as it is; and so is
// d·(z - 16), which makes the value one multiply-add of the f16 number 16 + code. A (page, head) of the pool is
// one piece: the codes of its positions, then their heads of blocks (an even number a position).
#ifndef BB_PAGED4_H
#define BB_PAGED4_H
#include <stddef.h>
#include <stdint.h>

namespace bb {

// Blocks' heads that a position has, bytes of a (page, head).
constexpr size_t kv4_heads(size_t hd) { return (hd / 32 + 1) / 2 * 2; }
constexpr size_t kv4_chunk(size_t page_size, size_t hd) {
  return (page_size * (hd / 2 + 2 * kv4_heads(hd)) + 15) / 16 * 16;
}

}  // namespace bb

#ifdef __HIPCC__
#include "bb_paged_device.h"
namespace bb {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// Where the head of block b of a page's position lies in its (page, head).
__device__ __forceinline__ int kv4_head_at(const PagedView& kv, int pos, int b) {
  return kv.page_size * (kv.hd / 2) + 2 * (pos * ((kv.hd / 32 + 1) & ~1) + b);
}

template <int N>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  typedef uint32_t V __attribute__((ext_vector_type(N), aligned(4 * N)));
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = v[i];
  }
}

// What 16 + code is made with: a constant that stands in a vector register, as an instruction with two of them needs.
struct Kv4Magic {
  uint32_t bits = 0x4c004c00u;  // 16 twice
  __device__ __forceinline__ Kv4Magic() { asm("" : "+v"(bits)); }
};
// The heads of two blocks (in the halves of a word), as what their codes are multiplied by and what is added.
struct Kv4Blocks {
  v2h d, zd;
  Kv4Blocks() = default;
  __device__ __forceinline__ explicit Kv4Blocks(uint32_t heads) {
    d = __builtin_bit_cast(v2h, heads & 0x7fc07fc0u);
    // 1024 + 64 + z, from the 6 lower bits and the sign turned round in the 7th
    const uint32_t low = (heads & 0x003f003fu) | 0x64006400u, sign = (heads ^ 0x80008000u) >> 9;
    const v2h z = __builtin_bit_cast(v2h, (sign & 0x00400040u) | (low & ~0x00400040u));
    zd = (z - v2h{(_Float16)1104.0f, (_Float16)1104.0f}) * d;
  }
  // One block twice.
  static __device__ __forceinline__ Kv4Blocks of(uint32_t head) { return Kv4Blocks(head | head << 16); }
  // The I-th half byte of both halves of a word as the elements they stand for.
  template <int I>
  __device__ __forceinline__ uint32_t pair(uint32_t w, const Kv4Magic& m) const {
    const uint32_t at = I == 0 ? w << 6 : I == 1 ? w << 2 : I == 2 ? w >> 2 : w >> 6;  // to bits 6 to 9 of each half
    const v2h x = __builtin_bit_cast(v2h, (at & 0x03c003c0u) | m.bits);                // 16 + code
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, d, zd));
  }
  // A word's 8 elements in their order, and in the order 0 4 1 5 2 6 3 7 (of one block twice).
  __device__ __forceinline__ v4u natural(uint32_t w, const Kv4Magic& m) const {
    const uint32_t a = pair<0>(w, m), b = pair<1>(w, m), c = pair<2>(w, m), e = pair<3>(w, m);
    return v4u{__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(e, c, 0x05040100u),
               __builtin_amdgcn_perm(b, a, 0x07060302u), __builtin_amdgcn_perm(e, c, 0x07060302u)};
  }
  __device__ __forceinline__ v4u paired(uint32_t w, const Kv4Magic& m) const {
    return v4u{pair<0>(w, m), pair<1>(w, m), pair<2>(w, m), pair<3>(w, m)};
  }
};

// Whether step d (at least 0) reaches from lo to hi in 15 steps, and each of them by the offsets there are. (In f64: the
// products are exact, and so is the difference but for values 2^28 times apart.)
__device__ __forceinline__ bool kv4_step_holds(float d, float lo, float hi) {
  return 15.0 * (double)d >= (double)hi - (double)lo && 63.0 * (double)d >= (double)hi && 47.0 * (double)d >= -(double)lo;
}
// The smallest step that holds: from the largest that the f32 quotients (off by 2^-22) reach, the next at most.
__device__ __forceinline__ float kv4_step(float lo, float hi) {
  constexpr float UNIT = 3.814697265625e-6f;  // 2^-18, of the steps below 2^-13
  const float r = fmaxf((hi - lo) * (1.0f / 15.0f), fmaxf(hi * (1.0f / 63.0f), lo * (-1.0f / 47.0f)));
  const float d = r < 6.103515625e-5f ? floorf(r * 262144.0f) * UNIT : as_float(__float_as_uint(r) & 0xfff80000u);
  if (kv4_step_holds(d, lo, hi)) return d;
  return d < 6.103515625e-5f ? d + UNIT : as_float(__float_as_uint(d) + 0x00080000u);
}
// Eight elements of a block, of which four adjacent lanes hold a quarter each, as a word of codes; `head` is the block's.
// x / d is x·r corrected once by its remainder, r = 1 / d rounded: that is the quotient rounded to f32. And rounded to f32
// and then to an integer it is x / d rounded to an integer: the borders (n + 1/2)·d, n below 64, are f32 numbers, so that an
// x which is not on one is at least 2^-24 of itself away, and a quotient's rounding moves it less than that towards one.
__device__ __forceinline__ float kv4_quotient(float x, float d, float r) {
  const float q = x * r;
  return rintf(fmaf(fmaf(-q, d, x), r, q));
}
// The lanes of four in another order: 0xb1 neighbours exchanged, 0x4e pairs.
template <int ORDER>
__device__ __forceinline__ uint32_t quad(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ORDER, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t kv4_quantise(float (&x)[8], uint32_t& head) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    odd |= !(fabsf(x[i]) < __builtin_inff());
    x[i] = __builtin_amdgcn_fmed3f(x[i], -16384.0f, 16384.0f);
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  uint32_t any = odd;
  lo = fminf(lo, as_float(quad<0xb1>(__float_as_uint(lo))));
  hi = fmaxf(hi, as_float(quad<0xb1>(__float_as_uint(hi))));
  any |= quad<0xb1>(any);
  lo = fminf(lo, as_float(quad<0x4e>(__float_as_uint(lo))));
  hi = fmaxf(hi, as_float(quad<0x4e>(__float_as_uint(hi))));
  any |= quad<0x4e>(any);
  if (any) {
    head = 0x7fc0u;
    return 0;
  }
  const float d = kv4_step(lo, hi);
  head = 0;
  if (d == 0.0f) return 0;
  const float r = 1.0f / d, zf = kv4_quotient(lo, d, r);
  const int z = (int)zf;
  head = __builtin_bit_cast(uint16_t, (_Float16)d) | (uint32_t)(z & 63) | (z < 0 ? 0x8000u : 0u);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w |= (uint32_t)__builtin_amdgcn_fmed3f(kv4_quotient(x[i], d, r) - zf, 0.0f, 15.0f) << 4 * i;
  return w;
}

}  // namespace
}  // namespace bb
#endif
#endif
