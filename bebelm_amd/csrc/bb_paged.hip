// bb_paged.hip — rotary positions, appending to a paged key/value cache, and attention of one new
// token per sequence over it (include/bebelm_moe.h states the operators). The reference has no
// counterpart: values are computed in f32 from the formulas and rounded once where they are stored.
#include "bb_device.h"
#include <algorithm>
#include "bb_internal.h"

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

// N consecutive elements (whole 16-byte pieces, or one element) as f32, and back, rounded to nearest.
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = (float)p[0];
  } else {
    constexpr int M = 16 / sizeof(T);
    typedef T V __attribute__((ext_vector_type(M)));
#pragma unroll
    for (int i = 0; i < N; i += M) {
      const V v = *reinterpret_cast<const V*>(p + i);
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
    constexpr int M = 16 / sizeof(T);
    typedef T V __attribute__((ext_vector_type(M)));
#pragma unroll
    for (int i = 0; i < N; i += M) {
      V v;
#pragma unroll
      for (int j = 0; j < M; ++j) v[j] = (T)x[i + j];
      *reinterpret_cast<V*>(p + i) = v;
    }
  }
}

// Where page `page` of sequence s starts in the pool, -1 for a page that is not there.
__device__ __forceinline__ int64_t page_base(const PagedView& kv, const PagedSeqs& sq, int s, int page) {
  if (page < 0 || page >= sq.max_pages) return -1;
  const int p = sq.table[(size_t)s * sq.table_stride + page];
  return p < 0 || p >= kv.n_pages ? -1 : (int64_t)((size_t)p * kv.page_stride);
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
constexpr int RR_TPB_MAX = 8;  // tokens of a block at most

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
  const int ix = (int)index, page = ix / kv.page_size;
  w.live = 1;
  w.pos = r.pos ? r.pos[t] : ix;
  if (r.n_kv) {
    const int64_t pb = page_base(kv, sq, s, page);
    if (pb >= 0) w.base = pb + (int64_t)((size_t)(ix - page * kv.page_size) * kv.pos_stride);
  }
  return w;
}

// A block takes tpb tokens. Its waves find the tokens' places, its threads the (cos, sin) of every
// (token, pair) once into LDS; then groups of gs lanes (a power of two) take the tokens' head rows, a
// lane two runs of VE elements that turn together (or one run past the turned part). VE 8: whole
// 16-byte pieces; VE 1: any size and stride.
template <class A, class C, int VE>
__global__ void __launch_bounds__(RR_THREADS) k_rope_rows(RopeRows r, RopeTurns rt, PagedView kv, PagedSeqs sq, int tpb,
                                                          int gs) {
  extern __shared__ float2 cs[];  // [tpb][half]
  __shared__ RowPlace place[RR_TPB_MAX];
  const int tid = threadIdx.x, half = rt.half;
  const size_t t0 = (size_t)blockIdx.x * tpb;
  for (int i = tid >> 6; i < tpb; i += RR_THREADS / 64) {
    const RowPlace w = row_place(r, kv, sq, t0 + i);
    if ((tid & 63) == 0) place[i] = w;
  }
  __syncthreads();
  for (int i = tid; i < tpb * half; i += RR_THREADS) {
    const float2 v = cos_sin_turns(place[i / half].pos, rt.turns[i % half]);
    cs[i] = make_float2(rt.magnitude * v.x, rt.magnitude * v.y);
  }
  __syncthreads();
  const int n_rows = r.n_q + 2 * r.n_kv, nu = half / VE, units = nu + (r.hd - 2 * half) / VE;
  const int lane = tid & (gs - 1);
  for (int i = tid / gs; i < tpb * n_rows; i += RR_THREADS / gs) {
    const int tk = i / n_rows, row = i - tk * n_rows;
    const RowPlace w = place[tk];
    const size_t t = t0 + tk;
    if (!w.live) continue;
    const bool is_q = row < r.n_q, is_k = !is_q && row < r.n_q + r.n_kv;
    if (!is_q && w.base < 0) continue;
    const int head = is_q ? row : is_k ? row - r.n_q : row - r.n_q - r.n_kv;
    const A* x = is_q   ? static_cast<const A*>(r.q) + t * r.q_ts + (size_t)head * r.q_hs
                 : is_k ? static_cast<const A*>(r.k) + t * r.k_ts + (size_t)head * r.hd
                        : static_cast<const A*>(r.v) + t * r.v_ts + (size_t)head * r.hd;
    A* yq = static_cast<A*>(r.q_out) + t * r.qo_ts + (size_t)head * r.qo_hs;
    C* yc = static_cast<C*>(is_k ? kv.k : kv.v) + w.base + (size_t)head * kv.head_stride;
    const float* gain = is_q ? r.q_norm : is_k ? r.k_norm : nullptr;
    float scale = 1.0f;
    if (gain) {
      // rmsnorm over the head: the lanes of the group hold parts of it
      float ss = 0.0f;
      for (int u = lane; u < units; u += gs) {
        const int e0 = u < nu ? (rt.interleaved ? 2 * u * VE : u * VE) : 2 * half + (u - nu) * VE;
        float a[VE];
        load_vec<A, VE>(x + e0, a);
#pragma unroll
        for (int j = 0; j < VE; ++j) ss += a[j] * a[j];
        if (u < nu) {
          load_vec<A, VE>(x + (rt.interleaved ? e0 + VE : e0 + half), a);
#pragma unroll
          for (int j = 0; j < VE; ++j) ss += a[j] * a[j];
        }
      }
      for (int o = 1; o < gs; o <<= 1) ss += __shfl_xor(ss, o);
      scale = 1.0f / sqrtf(ss / (float)r.hd + r.eps);
    }
    for (int u = lane; u < units; u += gs) {
      const bool turn = u < nu;
      const int e0 = turn ? (rt.interleaved ? 2 * u * VE : u * VE) : 2 * half + (u - nu) * VE;
      const int e1 = rt.interleaved ? e0 + VE : e0 + half;
      float a[VE], b[VE];
      load_vec<A, VE>(x + e0, a);
      if (turn) load_vec<A, VE>(x + e1, b);
      if (gain) {
#pragma unroll
        for (int j = 0; j < VE; ++j) a[j] = a[j] * scale * gain[e0 + j];
        if (turn)
#pragma unroll
          for (int j = 0; j < VE; ++j) b[j] = b[j] * scale * gain[e1 + j];
      }
      if (turn && (is_q || is_k)) {
        const float2* c = cs + tk * half + u * VE;
        if (rt.interleaved && VE > 1) {
          // pairs (0,1), (2,3), ... of the 2·VE elements a, b
#pragma unroll
          for (int j = 0; j < VE; j += 2) {
            const float2 ca = c[j / 2], cb = c[VE / 2 + j / 2];
            const float a0 = a[j], a1 = a[j + 1], b0 = b[j], b1 = b[j + 1];
            a[j] = a0 * ca.x - a1 * ca.y;
            a[j + 1] = a0 * ca.y + a1 * ca.x;
            b[j] = b0 * cb.x - b1 * cb.y;
            b[j + 1] = b0 * cb.y + b1 * cb.x;
          }
        } else {
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const float a0 = a[j], b0 = b[j];
            a[j] = a0 * c[j].x - b0 * c[j].y;
            b[j] = a0 * c[j].y + b0 * c[j].x;
          }
        }
      }
      if (is_q) {
        store_vec<A, VE>(yq + e0, a);
        if (turn) store_vec<A, VE>(yq + e1, b);
      } else {
        store_vec<C, VE>(yc + e0, a);
        if (turn) store_vec<C, VE>(yc + e1, b);
      }
    }
  }
}

template <class A, class C>
hipError_t rope_rows_of(hipStream_t s, const RopeRows& r, const RopeTurns& t, const PagedView& kv, const PagedSeqs& sq) {
  const size_t per = 16 / sizeof(A);
  // (arrays start 16-byte aligned, the pool's strides are whole 16-byte pieces)
  const bool wide = t.half % 8 == 0 && r.hd % 8 == 0 &&
                    (r.q_ts % per | r.q_hs % per | r.qo_ts % per | r.qo_hs % per | r.k_ts % per | r.v_ts % per) == 0;
  const int ve = wide ? 8 : 1, units = t.half / ve + (r.hd - 2 * t.half) / ve;
  int gs = 1;
  while (gs < units && gs < 64) gs *= 2;
  const int tpb = r.T >= 4096 ? 2 : 1;
  const dim3 grid((unsigned)((r.T + tpb - 1) / tpb));
  const size_t lds = (size_t)tpb * t.half * sizeof(float2);
  if (wide) BB_LAUNCH((k_rope_rows<A, C, 8>), grid, dim3(RR_THREADS), lds, s, r, t, kv, sq, tpb, gs);
  else BB_LAUNCH((k_rope_rows<A, C, 1>), grid, dim3(RR_THREADS), lds, s, r, t, kv, sq, tpb, gs);
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
namespace {

constexpr int PA_THREADS = 256;

// One block per (sequence, head): chunks of 256 positions, a thread a position's score, then a thread
// an element of the value sum; running maximum and sum over the chunks.
template <class A, class C>
__global__ void __launch_bounds__(PA_THREADS) k_paged_attn_rows(PagedQuery pq, PagedView kv, PagedSeqs sq) {
  __shared__ float q[OPS_HD_MAX], p[PA_THREADS], red[PA_THREADS / 64];
  __shared__ int64_t at[PA_THREADS];
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, hd = kv.hd;
  const int g = h / (pq.n_heads / kv.n_kv);
  const A* qr = static_cast<const A*>(pq.q) + (size_t)s * pq.q_stride + (size_t)h * hd;
  if (tid < hd) q[tid] = (float)qr[tid] * pq.scale;
  const int64_t cap = (int64_t)sq.max_pages * kv.page_size;
  const int len = (int)min((int64_t)max(sq.lens[s], 0), cap);
  const int first = pq.window > 0 ? max(0, len - pq.window) : 0;
  float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
  for (int j0 = first; j0 < len; j0 += PA_THREADS) {
    const int j = j0 + tid;
    int64_t e = -1;
    if (j < len) {
      const int page = j / kv.page_size;
      e = page_base(kv, sq, s, page);
      if (e >= 0) e += (int64_t)((size_t)(j - page * kv.page_size) * kv.pos_stride + (size_t)g * kv.head_stride);
    }
    __syncthreads();  // q is there; the chunk before is done with p and at
    float sc = -__builtin_inff();
    if (e >= 0) {
      const C* k = static_cast<const C*>(kv.k) + e;
      sc = 0.0f;
      for (int d = 0; d < hd; ++d) sc += q[d] * (float)k[d];
    }
    float mx = wave_max(sc);
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    at[tid] = e;
    __syncthreads();
    const float m1 = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float ms = m1 == -__builtin_inff() ? 0.0f : m1;
    p[tid] = e >= 0 ? expf(sc - ms) : 0.0f;
    const float f = expf(m - ms);
    m = m1;
    __syncthreads();
    l *= f;
    o *= f;
    for (int i = 0; i < min(PA_THREADS, len - j0); ++i) {
      if (at[i] < 0) continue;
      l += p[i];
      if (tid < hd) o += p[i] * (float)(static_cast<const C*>(kv.v) + at[i])[tid];
    }
  }
  const bool none = m == -__builtin_inff() && l == 0.0f;
  if (tid < hd) (static_cast<A*>(pq.out) + (size_t)s * pq.out_stride + (size_t)h * hd)[tid] = (A)(none ? 0.0f : o / l);
  if (tid == 0 && pq.lse) pq.lse[(size_t)s * pq.n_heads + h] = none ? m : m + logf(l);
}

}  // namespace

size_t paged_attn_ws(int, int, int, int, int) { return 0; }

hipError_t launch_paged_attn(hipStream_t s, int, int dtype, int cache, const PagedQuery& q, const PagedView& kv,
                             const PagedSeqs& seqs) {
  if (seqs.n_seqs == 0) return hipSuccess;
  return by_dtypes(dtype, cache, [&](auto a, auto c) {
    BB_LAUNCH((k_paged_attn_rows<typename decltype(a)::T, typename decltype(c)::T>), dim3(q.n_heads, seqs.n_seqs),
              dim3(PA_THREADS), 0, s, q, kv, seqs);
    return hipGetLastError();
  });
}

}  // namespace bb
