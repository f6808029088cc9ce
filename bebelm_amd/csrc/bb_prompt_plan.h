// bb_prompt_plan.h — how attention of several new tokens per sequence cuts its work: rows into tiles, the positions that
// a tile of rows sees into tiles of keys, these into parts for several blocks. Arithmetic only, shared by
// the kernels and their launch (bb_paged_prompt.hip); without HIP it is plain C++, which the host test runs.
#ifndef BB_PROMPT_PLAN_H
#define BB_PROMPT_PLAN_H
#include "bb_paged_plan.h"

namespace bb {

// The rows of a kv head: its G query heads of each of a sequence's n tokens (below 2^31 in all), `bm` a tile.
BB_BOTH int row_tiles(int n, int G, int bm) { return (int)(((int64_t)n * G + bm - 1) / bm); }
// Tiles of all sequences together, at most.
inline size_t most_tiles(size_t rows, int bm, size_t n_seqs) { return rows / bm + n_seqs < rows ? rows / bm + n_seqs : rows; }

// The tokens a sequence brings: seq_start's entries, whatever they hold, as a range of the call's tokens.
struct TokenSpan {
  int first, n;
};
BB_BOTH TokenSpan token_span(int from, int to, int n_tokens) {
  const int a = lesser(greater(from, 0), n_tokens), b = lesser(greater(to, 0), n_tokens);
  return {a, greater(b - a, 0)};
}

// The index of token t in its sequence (len and end as they come), held where its sums with a window stay 31 bits.
BB_BOTH int token_index(int len, int end, int t) {
  const int64_t i = (int64_t)len - end + t;
  return (int)(i < -1 ? -1 : i > 0x7ffffffe ? 0x7ffffffe : i);
}

// The first position that a token at index i sees behind the prefix.
BB_BOTH int first_seen(int i, int window) { return window > 0 ? greater(0, i - window + 1) : 0; }

// Tiles of kt positions that tokens at indexes i0..i1 of a sequence of len positions look at: the prefix's (0..head-1),
// then those of what the window leaves (from `from` on).
struct KeyTiles {
  int head, from, n;
  BB_BOTH int at(int u) const { return u < head ? u : u - head + from; }
};
BB_BOTH KeyTiles key_tiles(int i0, int i1, int len, int prefix, int window, int kt) {
  KeyTiles k;
  k.head = (lesser(prefix, len) + kt - 1) / kt;
  const int begin = first_seen(i0, window), end = lesser(len, i1 + 1);
  k.from = greater(begin / kt, k.head);
  k.n = k.head + (begin < end ? greater(0, (end + kt - 1) / kt - k.from) : 0);
  return k;
}

// n tiles in at most `most` parts of equal numbers, none (but the last) below `least`.
struct KeyParts {
  int per, used;
};
BB_BOTH KeyParts key_parts(int n, int most, int least) {
  KeyParts p;
  p.per = greater(least, (n + most - 1) / most);
  p.used = greater(1, (n + p.per - 1) / p.per);
  return p;
}

}  // namespace bb
#endif
