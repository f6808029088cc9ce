// bb_paged_prompt.hip — how attention of several new tokens per sequence is launched, and the sum of its parts; the kernels
// are in bb_paged_prompt.h.
#include "bb_paged_prompt.h"

namespace bb {

namespace {

// Adds the parts of rows, where there are several: `lanes` (16, 32 or 64) lanes a row, 4 elements each. Bound by its launch
// (4 to 5 us; its bytes, 512 rows of 8 heads of 64 in 4 parts, take 1).
__global__ void __launch_bounds__(PP_THREADS) k_prompt_join(PromptQuery pq, int hd, int bm, int lanes, PromptPlan pl, float up) {
  const int lane = threadIdx.x % lanes, in = (blockIdx.y * PP_THREADS + threadIdx.x) / lanes;
  const int4 at = pl.places[blockIdx.x];
  const int used = at.x, r = at.y + in;
  if (used <= 1 || in >= bm || r >= at.z) return;
  const size_t first = (size_t)blockIdx.x * pl.parts * bm + in;
  const int d = min(4 * lane, hd - 4);
  float m = NEG_INF, l = 0.0f;
  v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int p = 0; p < used; ++p) {
    const float2 ml = pl.ml[first + (size_t)p * bm];
    const v4f y = *reinterpret_cast<const v4f*>(pl.sums + (first + (size_t)p * bm) * hd + d);
    const float top = fmaxf(m, ml.x), ref = top == NEG_INF ? 0.0f : top;
    const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(ml.x - ref);
    m = top;
    l = l * f0 + ml.y * f1;
    x = x * f0 + y * f1;
  }
  const int t = at.w + r / pl.G, head = (int)(blockIdx.x % pl.n_kv) * pl.G + r % pl.G;
  const bool none = m == NEG_INF && l == 0.0f;
  if (4 * lane < hd)
    store_act(pq.out, (size_t)t * pq.out_stride + (size_t)head * hd + d, pq.dt, x * (none ? 0.0f : 1.0f / l));
  if (lane == 0 && pq.lse)
    pq.lse[(size_t)t * pq.n_heads + head] = none ? NEG_INF : (m + (__builtin_amdgcn_logf(l) - up)) * LN2;
}

constexpr int PARTS_MAX = 64;

// The blocks of a shape that a CU takes at once (0: it is not used).
int blocks_of_cu(int cache, int dt, int cls, int wr) {
  const auto blocks = [](auto s) { return decltype(s)::NEVER ? 0 : decltype(s)::WAVES; };
  return cache == BB_F32   ? shape_f32(dt, cls, wr, blocks)
         : cache == BB_F16 ? shape_f16(dt, cls, wr, blocks)
         : cache == BB_KV4 ? shape_kv4(dt, cls, wr, blocks)
                           : shape_bf16(dt, cls, wr, blocks);
}

// The blocks of a launch, chosen from what the host knows: how many tokens and sequences there are.
struct PromptCut {
  int wr;    // waves along a tile's rows: 4, or where there are few, its keys shared out to 4 / wr waves
  int bm, n_tiles, parts;
};
PromptCut prompt_cut(int n_cu, int cache, int dt, size_t n_tokens, size_t n_seqs, int G, int n_kv, int hd) {
  PromptCut c;
  const int cls = pa_class(hd);
  const size_t rows = n_tokens * (size_t)G, mean = (rows + n_seqs - 1) / n_seqs;
  // (16 x 12 tokens, 48 rows each, after 8192, heads of 128, bf16: 146, 114 and 122 us with tiles of 32, 64 and 128 rows; 8 x
  // 12 on an f32 cache, heads of 64: 110, 95 and 116; 16 x 5, 20 rows each, heads of 64, bf16: 53 and 62 with 32 and 64)
  c.wr = mean > 64 ? 4 : mean > 32 ? 2 : 1;
  while (blocks_of_cu(cache, dt, cls, c.wr) == 0) c.wr *= 2;  // (4 always is)
  c.bm = 32 * c.wr;
  c.n_tiles = (int)most_tiles(rows, c.bm, n_seqs);
  // keys in parts while the blocks (of sequences that are alike) fit the device at once (4 x 512 tokens after 2048, heads of
  // 128: 101 us, 109 in one part, 117 in twice as many; 200 after 8192: 52, 202 and 64; 16 x 5 after 1000: 24.3, 24.4 and 32)
  const size_t blocks = (mean + c.bm - 1) / c.bm * n_seqs * n_kv;
  const size_t at_once = (size_t)n_cu * blocks_of_cu(cache, dt, cls, c.wr);
  c.parts = (int)std::min<size_t>(PARTS_MAX, std::max<size_t>(1, at_once / blocks));
  return c;
}

size_t prompt_ws(const PromptCut& c, int n_kv, int hd) {
  if (c.parts == 1) return 0;
  const size_t tiles = (size_t)c.n_tiles * n_kv, slots = tiles * c.parts * c.bm;
  return slots * ((size_t)hd * 4 + sizeof(float2)) + tiles * sizeof(int4);
}

}  // namespace

size_t paged_prompt_ws(int n_cu, int cache, size_t n_tokens, size_t n_seqs, int n_heads, int n_kv, int hd) {
  size_t most = 0;
  if (n_tokens == 0 || n_seqs == 0) return 0;
  for (const int dt : {BB_F32, BB_F16, BB_BF16})
    most = std::max(most, prompt_ws(prompt_cut(n_cu, cache, dt, n_tokens, n_seqs, n_heads / n_kv, n_kv, hd), n_kv, hd));
  return most;
}

hipError_t launch_paged_prompt(hipStream_t st, int n_cu, int cache, const PromptQuery& q, const PagedView& kv,
                               const PagedSeqs& sq) {
  const int G = q.n_heads / kv.n_kv;
  const PromptCut c = prompt_cut(n_cu, cache, q.dt, q.n_tokens, sq.n_seqs, G, kv.n_kv, kv.hd);
  PromptPlan pl{G, c.n_tiles, kv.n_kv, c.parts, 1, false, nullptr, nullptr, nullptr};
  if (c.parts > 1) {
    const size_t tiles = (size_t)c.n_tiles * kv.n_kv, slots = tiles * c.parts * c.bm;
    pl.places = static_cast<int4*>(q.ws);
    pl.sums = reinterpret_cast<float*>(pl.places + tiles);
    pl.ml = reinterpret_cast<float2*>(pl.sums + slots * kv.hd);
  }
  const hipError_t e = cache == BB_F32   ? launch_prompt_f32(st, c.wr, q, kv, sq, pl)
                       : cache == BB_F16 ? launch_prompt_f16(st, c.wr, q, kv, sq, pl)
                       : cache == BB_KV4 ? launch_prompt_kv4(st, c.wr, q, kv, sq, pl)
                                         : launch_prompt_bf16(st, c.wr, q, kv, sq, pl);
  if (e != hipSuccess || pl.parts == 1) return e;
  const int lanes = pa_class(kv.hd) / 4;
  BB_LAUNCH(k_prompt_join, dim3(pl.n_tiles * pl.n_kv, c.bm * lanes / PP_THREADS), dim3(PP_THREADS), 0, st, q, kv.hd, c.bm,
            lanes, pl, cache == BB_F16 || cache == BB_KV4 ? F16_UP : 0.0f);
  return hipGetLastError();
}

}  // namespace bb
