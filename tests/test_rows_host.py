"""Whether two strided arrays share memory (csrc/bb_rows.h), compiled for the host, against every byte of theirs."""
import subprocess

from bebelm_amd import build

SOURCE = r'''
#include <cstdio>
#include <cstdint>
#include <random>
#include <set>
#include "%s/bb_rows.h"
using bb::Rows;

static std::set<uintptr_t> bytes(const Rows& r) {
  std::set<uintptr_t> s;
  for (size_t i = 0; i < r.n[0]; ++i)
    for (size_t j = 0; j < r.n[1]; ++j)
      for (size_t k = 0; k < r.len; ++k) s.insert((uintptr_t)r.p + i * r.stride[0] + j * r.stride[1] + k);
  return s;
}

int main() {
  std::mt19937 g(7);
  auto pick = [&](size_t lo, size_t hi) { return lo + g() %% (hi - lo + 1); };
  long meet = 0, apart = 0, missed = 0, refused = 0, odd = 0;
  for (int it = 0; it < 400000; ++it) {
    // the same strides for both (a group of either no longer than they are), or any
    const bool alike = it %% 4 != 0, nested = it %% 2 == 0;
    Rows r[2];
    const size_t s1 = pick(1, 12);
    for (auto& x : r) {
      x.n[0] = pick(1, 4);
      x.n[1] = pick(1, 4);
      x.len = pick(1, alike ? s1 : 12);
      x.stride[1] = alike ? s1 : pick(0, 12);
    }
    const size_t e = r[0].extent(1) > r[1].extent(1) ? r[0].extent(1) : r[1].extent(1);
    const size_t s0 = pick(e, e + 10);
    for (auto& x : r) x.stride[0] = alike ? s0 : pick(0, 40);
    if (alike && !nested) r[0] = bb::rows_of(nullptr, r[0].n[1], s1, r[0].len, 1), r[1] = bb::rows_of(nullptr, r[1].n[1], s1, r[1].len, 1);
    r[0].p = (const void*)(uintptr_t)1000;
    r[1].p = (const void*)(uintptr_t)pick(900, 1100);
    const auto a = bytes(r[0]), b = bytes(r[1]);
    bool want = false;
    for (uintptr_t x : a) want = want || b.count(x);
    const bool got = bb::rows_overlap(r[0], r[1]);
    odd += got != bb::rows_overlap(r[1], r[0]);
    missed += want && !got;
    refused += alike && got && !want;
    (want ? meet : apart) += 1;
  }
  std::printf("%%ld %%ld %%ld %%ld %%ld\n", missed, refused, odd, meet, apart);
}
'''


def test_rows_share_memory_exactly_where_a_byte_is_shared(tmp_path):
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(SOURCE % build.CSRC)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    missed, refused, odd, meet, apart = map(int, out.split())
    assert missed == 0, "arrays that share a byte pass for disjoint"
    assert refused == 0, "rows between each other pass for overlapping"
    assert odd == 0 and meet > 50_000 and apart > 50_000
