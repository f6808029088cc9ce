// bb_paged_plan.h — how attention over a paged cache cuts a batch into work: positions as slots of pages, units of
// slots, equal runs of units for the blocks, partial sums for the join. Arithmetic only, shared by the
// kernels and their launch (bb_paged.hip); without HIP it is plain C++, which the host test runs.
#ifndef BB_PAGED_PLAN_H
#define BB_PAGED_PLAN_H
#include <stddef.h>
#include <stdint.h>
#include <algorithm>

#ifdef __HIPCC__
#define BB_BOTH __host__ __device__ __forceinline__
#else
#define BB_BOTH inline
#endif

namespace bb {

BB_BOTH int lesser(int a, int b) { return a < b ? a : b; }
BB_BOTH int greater(int a, int b) { return a > b ? a : b; }

// ---- divisions -----------------------------------------------------------------------------------
// i / n for 0 <= i < 2^31: (i * mul) >> (31 + shift), mul = ceil(2^(31 + shift) / n), shift = ceil(log2(n)) (the
// product is off by less than i / 2^(31 + shift) < 1 / n).
struct SlotDivision {
  uint32_t mul;
  int shift;
};
inline SlotDivision slot_division(int n) {
  SlotDivision d{0, 0};
  while ((1 << d.shift) < n) ++d.shift;
  d.mul = (uint32_t)((((uint64_t)1 << (31 + d.shift)) + n - 1) / n);
  return d;
}
BB_BOTH int slot_quotient(int i, uint32_t mul, int shift) { return (int)(((uint64_t)(uint32_t)i * mul) >> (31 + shift)); }

// a / b for 0 <= a < 2^30, b >= 1, inv = 1 / b within 2^-22 of itself: two steps of an f32 quotient, each off by less
// than 2^-22 of itself and 1, then at most 1 off.
BB_BOTH int quotient_by(int a, int b, float inv) {
  int q = (int)((float)a * inv);
  q += (int)((float)(a - q * b) * inv);
  q -= q * b > a ? 1 : 0;
  q += (q + 1) * b <= a ? 1 : 0;
  return q;
}
// (the same for the wave on the device)
BB_BOTH int uniform_div(int a, int b) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_readfirstlane(quotient_by(a, b, __builtin_amdgcn_rcpf((float)b)));
#else
  return a / b;
#endif
}

// ---- pairs and units ------------------------------------------------------------------------------
// Positions of a unit (their logarithm): a 16-bit tile for each wave, two f32 ones. Of 64, 128 and 256, calls: 34
// sequences of up to 16384, bf16, 50.7, 41.2 and 42.0 us; one of 9001, 15.1, 13.7, 14.5; 7 of up to 3001, heads of
// 80, f16, 23.7, 20.8, 21.4; 2 of the last 100000, one kv head, 27.1, 25.9, 26.4; 64 of 8192, 368 each. f32 alone is
// a little faster with 64: 24 of up to 4096 with their append 26.4, 27.1, 28.3.
constexpr int PA_UNIT = 7;
// The same where no sequence can reach past one, by the table's width and the window (the launch knows no length):
// no pair is split and nothing is to be joined, which costs 4 to 5 us. By the bytes of a head's row (one sequence,
// 8 kv heads; whole and split): bf16, 64 elements: 512 positions 8.1 and 10.1 us, 1000 11.7 and 11.0; f32,
// 64: 512 10.4 and 10.9; f32, 256 elements (4 sequences): 256 17.9 and 19.1, 512 27.0 and 19.1.
constexpr int pa_unit_short(int row_bytes) { return row_bytes <= 256 ? 9 : 8; }
constexpr int PA_PAIR = 1;        // what a pair costs besides its units
constexpr int PA_HEADS = 16;      // heads of a group at most
// A pair of one tile is a wave's alone, and a pair of one unit where the block's run has this many of
// them: nothing is then joined, and a block is in four pairs at once. 168 sequences of up to 62, 16 kv
// heads of 256, 33 us (all waves on every pair: 58); 131 of up to 3, of 64, 8.4 and 13.6; 200 of up to
// 500, 8 heads of 128, 28 and 36.
constexpr int PA_ALONE = 2;
// From this average cost of a pair on, one block a CU works (the others end at once): its loads fill the
// memory's queues as well as four blocks' and disturb each other less. Batches of shorter pairs keep
// all the blocks that fit, which hide each other's beginnings and ends. One a CU and all, 8 kv heads:
// 64 sequences of 8192, 64 elements, bf16 191 and 199 us, f32 355 and 381; of 128, f16, 357 and 375; 100
// sequences of 2000, of 64, f16, 85 and 92; one of 9001, of 64, bf16, 13.7 and 15.8; 2 of 100000, one kv head of 128,
// 25.9 and 28.4. Up to 2000, 128 sequences, 16 heads of 64: 59 and 44; up to 700, 200 sequences, of 128: 50 and 41;
// 7 of up to 3001, 16 heads of 80, 22.4 and 20.8. Near the threshold the average (which knows neither how many pairs there
// are nor how unlike) misses by 4%: 34 of up to 16384 (18) 41.0 and 39.9; 24 of up to 4096, f32 (7) 26.1 and 27.2.
constexpr int PA_LONG = 16;

// Waves of a SIMD that fit: 128, 256, 512 registers each. (The forms with heads of up to 64 fill theirs: f32 queries on a
// bf16 cache and all 16-bit caches of odd pages spill 12 to 24 of them, capped or biased scores 2 to 30, at a pair's beginning
// and end; in the loop over tiles only 3, of f32 queries with such scores on a bf16 cache of odd pages. 4-bit tiles take fewer, and
// heads of 256 fit twice, but with f32 queries: 56 to 63 are spilled, 13 to 32 brought back for each tile, not measured
// against one wave; three waves with heads of 128, 64 sequences of 8192, 141 us, two 138.)
constexpr int pa_waves(int hdp, bool four = false) { return hdp == 64 ? 4 : hdp == 128 || four ? 2 : 1; }
constexpr int pa_class(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
inline int blocks_at_once(int n_cu, int hd, bool four = false) { return n_cu * pa_waves(pa_class(hd), four); }

// A kv head's G query heads: `split` groups of `hg` (the last may have fewer); n_groups of all kv heads.
struct HeadGroups {
  int G, split, hg, n_groups;
  // Whether a batch's units can be counted in 30 bits (cap: positions of a sequence at most; up to 3 slots for 2).
  bool fits(int n_seqs, size_t cap) const {
    return (size_t)n_seqs * (size_t)n_groups * ((3 * cap / 2 >> PA_UNIT) + 1 + PA_PAIR) < ((size_t)1 << 29);
  }
};
inline HeadGroups head_groups(int n_heads, int n_kv) {
  HeadGroups p;
  p.G = n_heads / n_kv;
  p.split = (p.G + PA_HEADS - 1) / PA_HEADS;
  p.hg = (p.G + p.split - 1) / p.split;
  p.n_groups = n_kv * p.split;
  return p;
}

// What is attended to of a sequence, positions counted as slots (a page as page_slots of them).
struct SeqSpan {
  int base, first, len, units;  // positions first..len-1, counted from base; units >= 1
};
BB_BOTH SeqSpan span_of(int raw_len, int page_size, int page_slots, int max_pages, int window, int unit) {
  SeqSpan r;
  r.len = lesser(greater(raw_len, 0), max_pages * page_size);
  r.first = window > 0 ? greater(0, r.len - window) : 0;
  const int empty = page_slots - page_size;
  if (empty > 0) {
    r.first += (int)((uint32_t)r.first / (uint32_t)page_size) * empty;
    r.len += r.len > 0 ? (int)((uint32_t)(r.len - 1) / (uint32_t)page_size) * empty : 0;
  }
  r.base = r.first & ~31;
  r.units = greater(1, (r.len - r.base + (1 << unit) - 1) >> unit);
  return r;
}

// ---- runs -----------------------------------------------------------------------------------------
// The cost of a block's run: `all` is what the sequences cost one group (units + PA_PAIR each).
BB_BOTH int run_cost(int all, int n_seqs, int n_groups, int grid, int few) {
  const int total = all * n_groups;
  if (all >= PA_LONG * n_seqs) grid = lesser(grid, few);
  return total <= grid ? 1 : uniform_div(total + grid - 1, grid);
}

// The units of a pair, whose cost begins at lo (the pair's own PA_PAIR first), that a run u..end-1 has.
struct PairPart {
  int first, units;  // units <= 0: none
};
BB_BOTH PairPart pair_part(int u, int end, int lo, int units) {
  const int begin = lo + PA_PAIR;
  PairPart p;
  p.first = greater(u - begin, 0);
  p.units = lesser(units, end - begin) - p.first;
  return p;
}

// Whether a wave takes the pair alone (kt: positions of a tile; left: the run's cost).
BB_BOTH bool pair_alone(int units, const SeqSpan& sp, int kt, int left) {
  return units == 1 && (sp.len - sp.base <= kt || left >= PA_ALONE * (1 + PA_PAIR));
}

// Where a block leaves the partial sum of a pair that is not whole in it: one that ends in it, one that begins there.
BB_BOTH size_t partial_slot(int block, bool begins) { return 2 * (size_t)block + (begins ? 1 : 0); }

// The blocks that have units of a pair.
struct PairBlocks {
  int first, last;
};
BB_BOTH PairBlocks pair_blocks(int lo, int cost, int chunk) {
  return {uniform_div(lo + PA_PAIR, chunk), uniform_div(lo + cost - 1, chunk)};
}

// ---- the launch -----------------------------------------------------------------------------------
struct PagedCut {
  bool uni;    // pages as whole 16 slots
  int slots;   // of a page
  int unit;    // the logarithm of a unit's slots
  int blocks;  // of the launch
  int few;     // blocks that work where pairs are long
  bool join;   // a pair may lie in several blocks
};
inline PagedCut paged_cut(int n_cu, int n_seqs, int n_groups, int page_size, size_t pos_stride, int max_pages, int window,
                          int hd, int elem_bytes) {
  PagedCut c;
  const size_t slots16 = ((size_t)page_size + 15) / 16 * 16;
  c.uni = 2 * slots16 <= 3 * (size_t)page_size && 16 * pos_stride < ((size_t)1 << 29);
  c.slots = c.uni ? (int)slots16 : page_size;
  // slots of a sequence that count, at most (a window begins anywhere in a page, and its slots anywhere in 32)
  size_t cap = (size_t)max_pages * c.slots;
  if (window > 0) {
    const size_t pages = ((size_t)window + page_size - 1) / page_size + 1;
    cap = std::min(cap, std::min((size_t)window + pages * (c.slots - page_size), pages * c.slots) + 31);
  }
  const int blocks_max = blocks_at_once(n_cu, hd, elem_bytes == 1), unit_short = pa_unit_short(hd * elem_bytes);
  // (4 bits want all the waves for their instructions: 64 sequences of 8192, heads of 128, 140 us and 178 with one block a CU,
  // of 64, 94 and 150)
  c.few = c.uni && elem_bytes > 1 ? n_cu : blocks_max;
  // (pairs of one unit take a block each at most, longer ones a block for each unit)
  c.unit = cap <= (size_t)1 << unit_short ? unit_short : PA_UNIT;
  const size_t pairs = (size_t)n_seqs * n_groups, units = ((cap - 1) >> c.unit) + 1;
  c.blocks = (int)std::min<size_t>(blocks_max, pairs * (units == 1 ? 1 : units + PA_PAIR));
  c.join = units > 1;
  return c;
}

}  // namespace bb
#endif
