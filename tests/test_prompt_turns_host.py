"""The order in which a block of prompt attention brings, reads and refills its tiles (csrc/bb_prompt_turns.h, which the
kernel runs), compiled for the host: each wave's reads and writes of LDS are noted with the number of barriers that it has
passed. What one wave writes and another reads or writes must have a barrier in between; so must what a wave has asked to be
brought and what it reads itself. Every reader must find what its tile's waves last wrote there."""
import subprocess

import pytest

from bebelm_amd import build

TURNS = r'''
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <vector>
#include "%s/bb_prompt_turns.h"
using namespace bb;

enum { KEYS, VALS, FLAGS, ODD };
struct Event {
  int wave, barrier, tile;  // tile: whose contents are read or written (-1: the waves' sums)
  bool write, late;         // late: asked for, there at the next landed()
};
// What happens to each (place, which of two, row), in the order of one wave after the other.
typedef std::map<int, std::vector<Event>> Memory;

struct Case {
  int n, waves_rows;              // tiles; waves along the rows (4, 2, 1)
  bool registers;                 // tiles that pass registers (4 bits, f32 parts)
  std::vector<int> shared, odd, past, far;  // by tile; odd: bit w: wave w's rows hold such values
};

struct Wave {
  const Case& c;
  Memory& mem;
  const int wv, wk, rows, own;    // rows of a tile, rows a wave brings
  int passed, asked, next, scored[2], weighed, looked, told_tile;
  bool wrong;

  Wave(const Case& c_, Memory& m, int w)
      : c(c_), mem(m), wv(w), wk(w %% (4 / c_.waves_rows)), rows(c_.waves_rows == 1 ? 128 : 64), own(rows / 4), passed(0),
        asked(-1), next(-1), scored{-1, -1}, weighed(-1), looked(-1), told_tile(-1), wrong(false) {}
  void at(int place, int two, int row, bool write, int tile, bool late = false) {
    mem[(place * 2 + two) * 1024 + row].push_back({wv, passed, tile, write, late});
  }
  int first() const { return 4 / c.waves_rows == 1 ? 0 : wk * 32; }
  int count() const { return 4 / c.waves_rows == 1 ? 64 : 32; }
  void tile(int place, int u, bool write, bool mine, bool late = false) {
    for (int r = 0; r < (mine ? own : count()); ++r) at(place, u & 1, (mine ? wv * own : first()) + r, write, u, late);
  }

  int found = -1;
  void find(int u) { found = u; }
  void keys(int u) {
    wrong |= found != u;
    asked = u;
    at(FLAGS, u & 1, wv, true, u);
    if (!c.registers) tile(KEYS, u, true, true, true);
  }
  void pass() { next = asked; }
  void values(int u) {
    wrong |= next != u;
    if (!c.registers) tile(VALS, u, true, true, true);
  }
  void put_keys(int u) { if (c.registers) tile(KEYS, u, true, true); }
  void put_values(int u) { if (c.registers) tile(VALS, u, true, true); }
  bool there = false;
  void landed() { there = true; }
  void barrier() { ++passed; }
  template <int I> void score(int u, Set<I>) {
    tile(KEYS, u, false, false);
    scored[I] = u;
  }
  template <int I> void see(int u, Set<I>) {
    wrong |= scored[I] != u;
    for (int w = 0; w < 4; ++w)   // (those whose rows the wave scores)
      if (w * own < first() + count() && (w + 1) * own > first()) at(FLAGS, u & 1, w, false, u);
  }
  template <int I, class F> void products(int u, Set<I>, F&& ask) {
    wrong |= scored[I] != u || weighed != u - 1;
    weighed = u;
    for (int j = 0; j < 4; ++j) {
      if (u + 1 < c.n) tile(KEYS, u + 1, false, false);
      ask(j);
    }
    if (u + 1 < c.n) tile(KEYS, u + 1, false, false);
    scored[1 - I] = u + 1;
    tile(VALS, u, false, false);
  }
  bool shared(int u) { return c.shared[u]; }
  bool odd(int u) {
    tile(VALS, u, false, true);
    looked = u;
    return c.odd[u] >> wv & 1;
  }
  void tell(int two, bool) {
    at(ODD, two, wv, true, looked);
  }
  bool told(int two) {
    for (int w = 0; w < 4; ++w) at(ODD, two, w, false, looked);
    return c.odd[looked] != 0;
  }
  void mark(int u) { tile(VALS, u, false, false); }
  void clean(int u) { tile(VALS, u, true, true); }
  void spoil(int) {}
  bool past() { wrong |= kept >= 0; return weighed + 1 < c.n && c.past[weighed + 1] >> wv & 1; }
  void raise() {}
  // (a maximum kept in a place of the wave's own while a turn is made; in set 0)
  int kept = -1;
  bool far() { return weighed + 1 < c.n && c.far[weighed + 1] >> wv & 1; }
  void near(int u) {
    wrong |= kept >= 0 || scored[0] != u;
    kept = u;
  }
  void back(int u) {
    wrong |= kept != u || weighed != u;
    kept = -1;
  }
  void last() { scored[0] = scored[1]; }
};

int main(int argc, char** argv) {
  std::mt19937 g(std::atoi(argv[1]));
  long races = 0, stale = 0, wrong = 0, cases = 0, looks = 0, plain = 0;
  for (int it = 0; it < 4000; ++it) {
    Case c{1 + (int)(g() %% 7), 1 << g() %% 3, (g() & 1) != 0, {}, {}, {}, {}};
    const int kind = g() %% 4;
    for (int u = 0; u < c.n; ++u) {
      c.shared.push_back(kind == 0 || (kind != 1 && (g() & 1)));
      c.odd.push_back(kind < 3 && g() %% 3 ? 0 : g() & 15);
      c.past.push_back(g() & 1 ? 0 : g() & 15);
      c.far.push_back(g() %% 3 ? 0 : g() & 15);
    }
    Memory mem;
    std::vector<int> passed;
    for (int w = 0; w < 4; ++w) {
      Wave wave(c, mem, w);
      PromptTurns<Wave>(wave, c.n).run();
      for (int two = 0; two < 2; ++two)
        for (int r = 0; r < wave.rows; ++r) wave.at(KEYS, two, r, true, -1), wave.at(VALS, two, r, true, -1);
      wrong += wave.wrong || wave.weighed != c.n - 1 || wave.kept >= 0 || !wave.there;
      passed.push_back(wave.passed);
    }
    for (int p : passed) wrong += p != passed[0];   // (a barrier that not all waves reach)
    for (const auto& m : mem) {
      const auto& e = m.second;
      for (size_t i = 0; i < e.size(); ++i)
        for (size_t j = i + 1; j < e.size(); ++j) {
          const Event &a = e[i], &b = e[j];
          if (a.barrier != b.barrier || (!a.write && !b.write) || (a.tile < 0 && b.tile < 0)) continue;
          // of one wave, in its order: only what it asked for and has not waited for
          races += a.wave != b.wave || (a.write && a.late);
        }
      // what a wave reads of a tile was written for it: the last writes before its barrier are that tile's
      for (const Event& r : e) {
        if (r.write) continue;
        const Event* w = nullptr;
        for (const Event& x : e)
          if (x.write && (x.barrier < r.barrier || (x.wave == r.wave && &x < &r)) && (!w || x.barrier >= w->barrier)) w = &x;
        stale += !w || w->tile != r.tile;
      }
    }
    ++cases;
    for (int u = 0; u < c.n; ++u) (c.shared[u] ? plain : looks) += 1;
  }
  std::printf("%%ld %%ld %%ld %%ld %%ld %%ld\n", races, stale, wrong, cases, looks, plain);
}
'''


@pytest.mark.parametrize("seed", range(2))
def test_waves_never_meet_at_a_tile(tmp_path, seed):
    src, exe = tmp_path / "turns.cpp", tmp_path / "turns"
    src.write_text(TURNS % build.CSRC)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wno-sign-compare", "-Wno-attributes", str(src), "-o", str(exe)],
                   check=True)
    races, stale, wrong, cases, looks, plain = map(int, subprocess.run(
        [str(exe), str(seed)], capture_output=True, text=True, check=True).stdout.split())
    assert (races, stale, wrong) == (0, 0, 0)
    assert cases == 4000 and looks > 1000 and plain > 1000
