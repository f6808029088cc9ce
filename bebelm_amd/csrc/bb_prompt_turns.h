// bb_prompt_turns.h — the order in which a block of k_paged_prompt (bb_paged_prompt.h) brings, scores and adds its tiles, and
// where its waves wait for each other. What a step does is the caller's (`B`): the kernel's, or the host test's, which
// notes what each wave reads and writes between two barriers. Without HIP it is plain C++.
#ifndef BB_PROMPT_TURNS_H
#define BB_PROMPT_TURNS_H

#define BB_INLINE __attribute__((always_inline))
#ifdef __HIPCC__
#define BB_TURN __device__ BB_INLINE
#else
#define BB_TURN
#endif

namespace bb {

// Turn u makes the scores of tile u + 1 while it weighs tile u, whose values it then adds, and asks for the keys of tile
// u + 2 and the values of tile u + 1. A tile's keys, values and flags (which of its rows are there) lie in the u & 1-th of two
// places each, and every wave brings some of a tile's rows. So what a turn refills has been read, by all waves, before the
// barrier that ended the turn before: keys and flags (tile u + 2's to tile u's place) in its products and in see(), values
// (tile u + 1's to tile u - 1's) when they were added. The first tile's scores are made before turn 0, which
// refills the place of its keys and flags: hence the barrier in begin().
//
// B's steps, of tile u: find(u), its rows in the page table; keys(u), asks for the rows found and notes which are there; pass(), the
// rows found last are those values(u) asks for next; put_keys(u), put_values(u), what came by way of registers goes to its place;
// landed(), what the wave asked for is there. score(u, set), see(u, set): scores into set u & 1, shaped and hidden;
// products(u, set, ask): tile u's scores weighed and its values added, tile u + 1's scores made, in between
// ask(0), ask(1), ask(2); shared(u): all rows of the block see all of the tile; odd(u): the wave brought values that
// are not finite, which tell() and told() make known to all; mark(u), clean(u), spoil(u): those taken out. past(): a
// score is past the running maximum's slack; raise(); far(): the maximum is too large for weights as they are made
// otherwise; near(u), back(u): before and after the turn of such scores. last(): the scores of set 1 become those of set 0.
template <int I>
struct Set {
  static constexpr int value = I;
};

template <class B>
struct PromptTurns {
  B& b;
  const int n;
  bool odd;
  int looks;
  BB_TURN PromptTurns(B& b_, int n_) : b(b_), n(n_), odd(false), looks(0) {}

  // Values that are not finite reach the rows that see them and no others. A tile that all rows of the block see is added
  // as it is; one that they do not is looked at when it is there. If it has such values, the sums
  // that they belong to are marked, the values taken out, and what is marked made NaN after the tile's turn.
  BB_TURN void look(int u) {
    if (b.shared(u)) return;
    const int at = looks++ & 1;  // (two places in turn: a wave that writes one again has passed a barrier behind its reads)
    b.tell(at, b.odd(u));
    b.barrier();
    odd = b.told(at);
  }

  template <int I>
  BB_TURN void turn(int u, Set<I> set) {
    const bool more = u + 1 < n, two = u + 2 < n;
    b.products(u, set, [&](int j) BB_INLINE {  // (behind the products of a step, which go on meanwhile)
      if (j == 0 && two) b.keys(u + 2);
      if (j == 1 && more) b.values(u + 1);
      if (j == 2 && two) {
        b.pass();
        if (u + 3 < n) b.find(u + 3);
      }
    });
    if (!more) return;
    b.see(u + 1, Set<1 - I>());
    if (two) b.put_keys(u + 2);
    b.put_values(u + 1);
    b.landed();
    b.barrier();
    look(u + 1);
  }

  // Tiles 0 and 1 on their way, the first's scores.
  BB_TURN void begin() {
    b.find(0);
    b.keys(0);
    b.pass();
    b.values(0);
    b.put_keys(0);
    b.put_values(0);
    if (n > 1) {
      b.find(1);
      b.keys(1);
      b.pass();
      b.put_keys(1);
      if (n > 2) b.find(2);
    }
    b.landed();
    b.barrier();
    b.score(0, Set<0>());
    b.see(0, Set<0>());
    b.barrier();  // (turn 0 refills their place, and look() need not wait)
    look(0);
  }

  // All of them (n > 0). What is seldom done to the sums stands outside the loop over plain turns, which keeps them in their
  // registers.
  BB_TURN void run() {
    begin();
    for (int u = 0; u < n;) {
      if (b.past()) b.raise();
      const bool far = b.far();
      if (far) b.near(u);
      if (odd) {
        b.mark(u);
        b.barrier();
        b.clean(u);
        b.barrier();
      }
      const bool spoiled = odd;
      odd = false;
      const auto on = [&]() BB_INLINE { return u < n && !spoiled && !far && !odd && !b.past(); };
      for (;;) {
        turn(u++, Set<0>());
        if (!on()) {
          b.last();
          break;
        }
        turn(u++, Set<1>());
        if (!on()) break;
      }
      if (spoiled) b.spoil(u - 1);
      if (far) b.back(u - 1);
    }
    b.barrier();  // (the tiles' place is taken behind it)
  }
};

}  // namespace bb
#endif
