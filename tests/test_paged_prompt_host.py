"""The host side of attention of several new tokens per sequence and of the 4-bit pool, without a GPU. The arithmetic by
which the former cuts its work (csrc/bb_prompt_plan.h, which the kernels and their launch include), compiled
for the host: tokens of a sequence whatever its entries hold, tiles that hold every position a row sees exactly once,
parts that are all of the tiles. How attention of single tokens cuts a 4-bit pool. The argument records and
the checks of the Python entry points."""
import struct
import subprocess

import numpy as np
import pytest
import torch

from bebelm_amd import _lib, build, kernels
from bebelm_amd.model import PagedKv
from test_paged_plan_host import RUNS

PLAN = r'''
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>
#include "%s/bb_prompt_plan.h"
using namespace bb;

int main(int argc, char** argv) {
  std::mt19937_64 g(std::atoi(argv[1]));
  auto pick = [&](int64_t lo, int64_t hi) { return (int)(lo + (int64_t)(g() %% (uint64_t)(hi - lo + 1))); };
  auto any = [&](std::vector<int> v) { return v[pick(0, (int64_t)v.size() - 1)]; };
  const int low = -2147483647 - 1, top = 2147483647;
  long bad[7] = {0}, seen[6] = {0};

  // spans lie in the call's tokens and are the entries' own where these are right
  for (int it = 0; it < 20000; ++it) {
    const int n = any({1, 2, 7, 500}), a = any({0, low, top, -1, n, n + 1, pick(0, n)}), b = any({0, low, top, -1, n, n + 1, pick(0, n)});
    const TokenSpan s = token_span(a, b, n);
    bad[0] += s.n < 0 || s.first < 0 || s.first > n || s.first + s.n > n;
    if (a >= 0 && a <= b && b <= n) bad[0] += s.first != a || s.n != b - a;
    // an index stays where sums with a window do not overflow, and is the difference where that is in range
    const int len = any({0, 1, top, pick(0, top), pick(0, 100)}), end = any({low, top, 0, n, pick(0, n)}), t = pick(0, 4194303);
    const int i = token_index(len, end, t);
    const int64_t exact = (int64_t)len - end + t;
    bad[1] += i < -1 || i == top || (exact >= -1 && exact < top && i != exact) || (exact < -1 && i != -1);
    const int w = any({0, 1, 2, top, pick(1, 1000)}), f = first_seen(i, w);
    bad[1] += f < 0 || (w == 0 ? f != 0 : f != (int)std::max<int64_t>(0, (int64_t)i - w + 1));
  }

  // sequences' tiles are no more than what the launch has
  for (int it = 0; it < 2000; ++it) {
    const int G = any({1, 2, 7, 16, 33}), bm = any({32, 64, 128}), n_seqs = pick(1, 40);
    size_t rows = 0, tiles = 0;
    for (int s = 0; s < n_seqs; ++s) {
      const int n = any({0, 0, 1, 1, 2, 31, 32, 33, 128, pick(0, 700)});
      rows += (size_t)n * G;
      tiles += row_tiles(n, G, bm);
      bad[2] += (int64_t)row_tiles(n, G, bm) * bm < (int64_t)n * G || ((int64_t)row_tiles(n, G, bm) - 1) * bm >= std::max(1, n * G);
    }
    bad[2] += tiles > most_tiles(rows, bm, n_seqs);
    seen[0] += tiles == most_tiles(rows, bm, n_seqs);
  }
  bad[2] += row_tiles(4194303, 511, 32) != (int)((4194303ll * 511 + 31) / 32);

  // every position that a token between the first and the last sees lies in one tile, and none comes twice
  for (int it = 0; it < 4000; ++it) {
    const int len = any({1, 2, 31, 32, 33, 127, 128, 129, pick(1, 900)}), n = pick(1, std::min(len, 70));
    const int kt = any({32, 64, 128}), window = any({0, 0, 1, 2, 31, 32, 33, 64, 65, 200, 5000}), prefix = any({0, 0, 1, 31, 32, 33, len, pick(0, len)});
    const int t1 = pick(0, n - 1), t0 = pick(0, t1);
    const int i0 = token_index(len, n, t0), i1 = token_index(len, n, t1);
    const KeyTiles k = key_tiles(i0, i1, len, prefix, window, kt);
    std::set<int> tiles;
    for (int u = 0; u < k.n; ++u) bad[3] += !tiles.insert(k.at(u)).second || k.at(u) < 0 || (int64_t)k.at(u) * kt >= len;
    for (int t = t0; t <= t1; ++t) {
      const int i = token_index(len, n, t);
      for (int j = 0; j < len; ++j)
        if ((j <= i && j >= first_seen(i, window)) || j < prefix) bad[4] += !tiles.count(j / kt);
    }
    // and no tile is there that nothing of the span sees
    for (const int u : tiles) {
      const int a = u * kt, b = std::min(len, a + kt) - 1;
      bad[5] += !(a < prefix || (a <= i1 && b >= first_seen(i0, window)));
    }
    seen[1] += prefix > 0 && window > 0 && k.from > k.head;
    seen[2] += k.n == 0;
    seen[2] += k.n == 1;
  }

  // parts are all of the tiles in order, none empty, no smaller than the least but the last
  for (int it = 0; it < 20000; ++it) {
    const int n = any({0, 1, 2, 3, 7, 64, pick(0, 5000)}), most = pick(1, 64), least = any({1, 2, 4, 8});
    const KeyParts p = key_parts(n, most, least);
    int at = 0;
    for (int i = 0; i < p.used; ++i) {
      const int u0 = i * p.per, u1 = std::min(n, u0 + p.per);
      bad[6] += u0 != at || (n > 0 && u1 <= u0) || (i + 1 < p.used && u1 - u0 < least);
      at = u1;
    }
    bad[6] += at != n || p.used < 1 || p.used > most;
    seen[3] += p.used == most && most > 1;
    seen[4] += p.used > 1 && p.used < most;
    seen[5] += n == 0;
  }
  for (long b : bad) std::printf("%%ld ", b);
  for (long s : seen) std::printf("%%ld ", s);
  std::printf("\n");
}
'''


@pytest.mark.parametrize("seed", range(4))
def test_prompt_plan(tmp_path, seed):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PLAN % build.CSRC)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wno-sign-compare", "-ftrapv",
                    str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe), str(seed)], capture_output=True, text=True, check=True).stdout.split()))
    what = ("spans", "indexes", "tiles of rows", "tiles that come twice", "positions in no tile", "tiles for nothing", "parts")
    assert got[:7] == [0] * 7, {w: n for w, n in zip(what, got[:7]) if n}
    assert min(got[7:]) > 10, "a part of the rules was hardly reached: %s" % got[7:]


@pytest.mark.parametrize("seed", range(2))
def test_runs_over_4_bits(tmp_path, seed):
    """The runs of blocks of tests/test_paged_plan_host.py, for pools whose head sizes are whole blocks of 32."""
    source = RUNS
    for was, now in (("hd = 8 * pick(1, 32), eb = any({2, 4})", "hd = 32 * pick(1, 8), eb = any({1})"),
                     ("blocks_at_once(n_cu, hd)", "blocks_at_once(n_cu, hd, true)")):
        assert was in source
        source = source.replace(was, now)
    src, exe = tmp_path / "runs.cpp", tmp_path / "runs"
    src.write_text(source % build.CSRC)
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-Wall", "-Wno-sign-compare", str(src), "-o", str(exe)],
                   check=True)
    got = list(map(int, subprocess.run([str(exe), str(seed)], capture_output=True, text=True, check=True).stdout.split()))
    assert got[:8] == [0] * 8
    assert min(got[8:14]) > 20


def test_argument_records_match_the_header(tmp_path):
    records = {"bb_paged_rows": (_lib.PAGED_ROWS, "seq_start"), "bb_paged_queries": (_lib.PAGED_QUERIES, "workspace_bytes")}
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(void) {\n%s return 0; }\n' % (
        _lib.HEADER, "".join(f'  printf("{n} %zu %zu\\n", sizeof({n}), offsetof({n}, {f}));\n' for n, (_, f) in records.items())))
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, size, off = line.split()
        record = records[name][0]
        assert record.size == int(size)
        assert struct.calcsize(record.format[:-1]) <= int(off) == int(size) - 8


class NoGpu:
    """A context that no call may reach."""
    handle, device = None, 0


class Pool:
    handle, n_kv_heads, head_dim = None, 2, 64


def test_python_checks():
    table, lens, start = np.zeros((3, 2), np.int32), np.ones(3, np.int32), np.array([0, 2, 2, 5], np.int32)
    q = np.zeros((5, 4, 64), np.float32)
    for kw in (dict(out=q[:3]), dict(out=q.astype(np.float16)), dict(q=q[:, :, :32]), dict(q=q.astype(np.float64)),
               dict(q=q[:, :, ::2]), dict(scale=0.0), dict(window=-1), dict(lse=np.zeros((3, 4), np.float32)),
               dict(lse=np.zeros((5, 4), np.float16)), dict(slopes=np.zeros(2, np.float32)), dict(slopes=np.zeros(4)),
               dict(prefix=np.zeros(5, np.int32)), dict(prefix=np.zeros(3, np.int64)), dict(seq_start=start[:3]),
               dict(seq_start=start.astype(np.int64)), dict(lens=lens[:2]), dict(table=table.astype(np.int64)),
               dict(table=table[0]),
               dict(workspace=np.zeros(1 << 20, np.uint8)), dict(workspace=torch.zeros(1 << 20))):
        a = dict(table=table, lens=lens, q=q, out=q.copy(), seq_start=start) | kw
        with pytest.raises(ValueError):
            kernels.paged_prompt_attention(NoGpu, Pool, a.pop("table"), a.pop("lens"), a.pop("q"), a.pop("out"), **a)
    rows = np.zeros((5, 2, 64), np.float32)
    for kw in (dict(k=None, v=None), dict(v=rows[:3]), dict(v=rows.astype(np.float16)), dict(k=rows.astype(np.int32)),
               dict(k=rows[:, :, :32]), dict(k=rows[:, ::2]), dict(seq_start=start[:3]), dict(lens=lens[:2])):
        a = dict(table=table, lens=lens, k=rows.copy(), v=rows.copy(), seq_start=start) | kw
        with pytest.raises(ValueError):
            kernels.paged_read(NoGpu, Pool, a.pop("table"), a.pop("lens"), **a)


def test_4_bit_pools_over_tensors():
    # (32 elements are 16 bytes of codes and 2 of their step and offset; a page's bytes end on whole 16)
    size = 16 * (2 * 16 + 2 * 2)
    k = torch.zeros(4, 2, size, dtype=torch.uint8)
    for args in ((k, k[:2], 16, 64), (k, k[:, :, :-1], 16, 64), (k, k, 8, 64), (k.float(), k.float(), 16, 64),
                 (k[0], k[0], 16, 64), (k, k, 16, 64)):   # (the last: not the context's GPU)
        with pytest.raises(ValueError):
            PagedKv.four_bit(NoGpu, *args)
