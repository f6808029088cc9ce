// bb_paged_device.h — what the kernels of the paged cache share: elements of its types as f32 and back, pages of
// positions, values as sums of 16-bit parts, sums over a wave.
#ifndef BB_PAGED_DEVICE_H
#define BB_PAGED_DEVICE_H
#include "bb_device.h"
#include <type_traits>
#include "bb_internal.h"
#include "bb_paged_plan.h"

namespace bb {
namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float NEG_INF = -__builtin_inff();

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

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

// cap·tanh(s / cap) of a score s (base 2), within a few units in the last place of itself whatever the cap. With y = s / cap, up
// to 0.6, s times a quotient of polynomials (tanh(y) / y by the continued fraction
// 1 / (1 + y^2 / (3 + y^2 / (5 + y^2 / (7 + y^2 / 9)))), off by less than 1e-9 there), then cap·(e - 1) / (e + 1),
// e = exp(2|y|). (Past a cap of 2.3e38, base 2's largest number stands for it.)
__device__ __forceinline__ float capped(float s, const ScoreCap& cap) {
  const float y = s * cap.inv, a = fabsf(y), z = y * y;
  const float e = __builtin_amdgcn_exp2f((a > 15.0f ? 15.0f : a) * (2.0f * LOG2E));
  const bool small = a < 0.6f;
  float n0 = fmaf(z, 105.0f + z, 945.0f), d0 = fmaf(z, fmaf(z, 15.0f, 420.0f), 945.0f), n1 = e - 1.0f, d1 = e + 1.0f;
  // (both in line: a branch each would cost more; and not done where a call has no cap)
  asm volatile("" : "+v"(n0), "+v"(d0), "+v"(n1), "+v"(d1));
  const float num = small ? n0 : n1, den = small ? d0 : d1;
  return (small ? s : copysignf(cap.top, s)) * (num * __builtin_amdgcn_rcpf(den));
}

}  // namespace
}  // namespace bb
#endif
