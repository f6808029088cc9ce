"""The arithmetic by which paged attention cuts a batch (csrc/bb_paged_plan.h, which the kernels and their launch include),
compiled for the host: divisions, slots, runs of blocks that cover every position once, and partial sums
where the join looks for them."""
import subprocess

import pytest

from bebelm_amd import build

DIVISIONS = r'''
#include <cmath>
#include <cstdio>
#include <random>
#include "%s/bb_paged_plan.h"
using namespace bb;

int main() {
  std::mt19937_64 g(3);
  auto pick = [&](uint64_t lo, uint64_t hi) { return lo + g() %% (hi - lo + 1); };
  long bad_quotient = 0, bad_slot = 0;
  for (int it = 0; it < 3000000; ++it) {
    const int b = (int)(1 + pick(0, (1ull << pick(1, 30)) - 2)), k = (int)pick(0, ((1 << 30) - 1) / b);
    const int64_t a64 = (int64_t)k * b + (it %% 4 == 0 ? 0 : it %% 4 == 1 ? b - 1 : (int64_t)pick(0, b - 1));
    if (a64 >= 1 << 30) continue;
    const int a = (int)a64;
    float inv = 1.0f / (float)b;   // (and what an approximate reciprocal may give)
    if (it %% 3) inv = std::nextafter(inv, it %% 3 == 1 ? 0.0f : 2.0f);
    bad_quotient += quotient_by(a, b, inv) != a / b;
  }
  for (int it = 0; it < 6000; ++it) {
    const int n = it < 3000 ? it + 1 : (int)pick(1, (1 << 20) + 15);
    const SlotDivision d = slot_division(n);
    const int64_t top = ((int64_t)1 << 31) - 1;
    for (int j = 0; j < 40; ++j) {
      const int64_t i = j < 2 ? j : j == 2 ? n - 1 : j == 3 ? n : j == 4 ? top : j == 5 ? top / n * n : j == 6 ? top / n * n - 1
                        : j < 20 ? (int64_t)pick(0, top / n) * n - (int64_t)pick(0, 1) : (int64_t)pick(0, top);
      if (i >= 0 && i <= top) bad_slot += slot_quotient((int)i, d.mul, d.shift) != i / n;
    }
  }
  std::printf("%%ld %%ld\n", bad_quotient, bad_slot);
}
'''

RUNS = r'''
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <vector>
#include "%s/bb_paged_plan.h"
using namespace bb;

int main(int argc, char** argv) {
  std::mt19937_64 g(std::atoi(argv[1]));
  auto pick = [&](int64_t lo, int64_t hi) { return (int)(lo + (int64_t)(g() %% (uint64_t)(hi - lo + 1))); };
  auto any = [&](std::vector<int> v) { return v[pick(0, (int64_t)v.size() - 1)]; };
  long bad[8] = {0}, seen[8] = {0};
  for (int it = 0; it < 1500; ++it) {
    const int page = any({1, 3, 5, 8, 10, 11, 12, 13, 16, 17, 21, 24, 33, 40, 64, 100, 256}), hd = 8 * pick(1, 32), eb = any({2, 4});
    const int n_kv = any({1, 2, 3, 8}), G = any({1, 2, 4, 7, 16, 17, 33}), n_cu = any({1, 3, 8, 256});
    const int n_seqs = any({1, 1, 2, 5, 12, 40}), max_pages = pick(1, any({1, 4, 40, 400}));
    const int cap = page * max_pages, window = any({0, 0, 1, 31, 32, 33, 100, 1000, 40000, pick(200, 256), pick(450, 512)});
    const HeadGroups hg = head_groups(n_kv * G, n_kv);
    const size_t pos_stride = it %% 50 == 0 ? (size_t)1 << 25 : 512;
    const PagedCut cut = paged_cut(n_cu, n_seqs, hg.n_groups, page, pos_stride, max_pages, window, hd, eb);
    seen[0] += cut.uni;
    seen[1] += !cut.uni;
    seen[2] += cut.join;
    seen[3] += !cut.join;
    // the groups of a kv head hold each of its heads once
    int heads = 0;
    for (int sub = 0; sub < hg.split; ++sub) heads += std::max(0, std::min(hg.hg, hg.G - sub * hg.hg));
    bad[0] += heads != hg.G || hg.hg > PA_HEADS || hg.G - (hg.split - 1) * hg.hg < 1;

    const auto slot = [&](int p) { return p + p / page * (cut.slots - page); };
    std::vector<SeqSpan> sp;
    std::vector<int> before{0};
    for (int s = 0; s < n_seqs; ++s) {
      const int n = any({0, 1, -1, cap, cap + 5, pick(0, cap), pick(0, cap), pick(0, std::min(cap, 40))});
      sp.push_back(span_of(n, page, cut.slots, max_pages, window, cut.unit));
      const SeqSpan& r = sp.back();
      // exactly the slots of the positions attended to lie in first..len-1
      const int len = std::min(std::max(n, 0), cap), first = window > 0 ? std::max(0, len - window) : 0;
      bad[1] += len > first && (r.first != slot(first) || r.len != slot(len - 1) + 1);
      bad[1] += r.base > r.first || r.base %% 16 || r.first - r.base > 31 || r.units != std::max(1, (r.len - r.base + (1 << cut.unit) - 1) >> cut.unit);
      bad[2] += !cut.join && r.units != 1;
      before.push_back(before.back() + r.units + PA_PAIR);
    }
    // as the blocks of the launch go through them
    const int all = before.back(), total = all * hg.n_groups, grid = cut.blocks;
    const int chunk = run_cost(all, n_seqs, hg.n_groups, grid, cut.few);
    bad[3] += hg.fits(n_seqs, (size_t)cap) ? total >= 1 << 30 : 1;
    bad[3] += grid < 1 || grid > blocks_at_once(n_cu, hd);
    std::map<std::pair<int, int>, std::vector<std::pair<int, int>>> got;
    std::map<std::pair<int, int>, std::vector<size_t>> parts;
    std::set<size_t> used;
    int working = 0;
    for (int block = 0; block < grid && (int64_t)block * chunk < total; ++block, ++working) {
      const int u = block * chunk, end = std::min(u + chunk, total);
      int s = 0;
      while (before[s + 1] * hg.n_groups <= u) ++s;
      int cost = before[s + 1] - before[s], grp = (u - before[s] * hg.n_groups) / cost;
      for (int lo = before[s] * hg.n_groups + grp * cost; lo < end; lo += cost, ++grp) {
        if (grp == hg.n_groups) grp = 0, ++s, cost = before[s + 1] - before[s];
        const int nu = cost - PA_PAIR;
        const PairPart p = pair_part(u, end, lo, nu);
        if (p.units <= 0) continue;
        const bool alone = pair_alone(nu, sp[s], eb == 4 ? 16 : 32, end - u);
        seen[4] += alone;
        bad[4] += alone && p.units != nu;
        const int k0 = sp[s].base + (p.first << cut.unit);
        got[{s, grp}].push_back({k0, std::min(k0 + (p.units << cut.unit), sp[s].len)});
        if (p.units != nu) {
          const size_t at = partial_slot(block, p.first == 0);
          bad[5] += !used.insert(at).second || at >= 2 * (size_t)blocks_at_once(n_cu, hd) || !cut.join;
          parts[{s, grp}].push_back(at);
          ++seen[5];
        }
      }
    }
    seen[6] += working < grid && total > grid;
    for (int s = 0; s < n_seqs; ++s)
      for (int grp = 0; grp < hg.n_groups; ++grp) {
        int at = sp[s].base;
        for (const auto& r : got[{s, grp}]) bad[6] += r.first != at, at = r.second;
        bad[6] += at != std::max(sp[s].len, sp[s].base) || got[{s, grp}].empty();
        // the join's view
        const int cost = before[s + 1] - before[s];
        const PairBlocks b = pair_blocks(before[s] * hg.n_groups + grp * cost, cost, chunk);
        std::vector<size_t> want;
        if (b.first != b.last)
          for (int i = b.first; i <= b.last; ++i) want.push_back(partial_slot(i, i == b.first));
        bad[7] += parts[{s, grp}] != want;
        seen[7] += want.size() > 2;
      }
  }
  for (long b : bad) std::printf("%%ld ", b);
  for (long s : seen) std::printf("%%ld ", s);
  std::printf("\n");
}
'''


def compiled(tmp_path, source, *args):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(source % build.CSRC)
    # (f32 products rounded one by one, as the kernels are built)
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-Wall", "-Wno-sign-compare", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, check=True).stdout
    return list(map(int, out.split()))


def test_divisions(tmp_path):
    assert compiled(tmp_path, DIVISIONS) == [0, 0]


@pytest.mark.parametrize("seed", range(4))
def test_runs(tmp_path, seed):
    got = compiled(tmp_path, RUNS, seed)
    what = ("head groups", "spans", "pairs split where nothing joins them", "counts", "split pairs of one wave",
            "places of partial sums", "positions", "the join's blocks")
    assert got[:8] == [0] * 8, {w: n for w, n in zip(what, got[:8]) if n}
    assert min(got[8:]) > 20, "a part of the rules was hardly reached: %s" % got[8:]
