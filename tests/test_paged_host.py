"""The host side of the paged-cache operators, without a GPU: how attention cuts a batch into runs of
blocks (every position once, partial sums where the join looks for them), the division that finds a
position's page, the argument records' layout, and the checks of the Python entry points."""
import random
import struct
import subprocess

import numpy as np
import pytest
import torch

from bebelm_amd import _lib, kernels

PAIR = 1   # what a pair costs besides its units


def slots(p, page):
    """A position as a slot: pages counted as whole 16 positions."""
    return p + p // page * (-(-page // 16) * 16 - page)


def span(n, cap, window, page, unit):
    n = min(max(n, 0), cap)
    first = max(0, n - window) if window else 0
    end, first = (slots(n - 1, page) + 1 if n else 0), slots(first, page)
    base = first & ~31
    return base, first, end, max(1, -(-(end - base) // unit))


def runs(lens, cap, window, page, groups, grid, unit):
    """{(sequence, group): slot ranges in order}, {(sequence, group): where its partial sums lie}, the
    costs of a group of each sequence, a run's cost: as k_paged_attn's blocks find them."""
    spans = [span(n, cap, window, page, unit) for n in lens]
    cost = [s[3] + PAIR for s in spans]
    total = sum(cost) * groups
    chunk = 1 if total <= grid else -(-total // grid)
    ranges, parts = {}, {}
    for block in range(grid):
        u = block * chunk
        end = min(u + chunk, total)
        if u >= total:
            break
        before = s = 0
        while (before + cost[s]) * groups <= u:
            before += cost[s]
            s += 1
        grp = (u - before * groups) // cost[s]
        lo = before * groups + grp * cost[s]
        while lo < end:
            if grp == groups:
                grp, s = 0, s + 1
            nu, first = cost[s] - PAIR, lo + PAIR
            u0 = max(u - first, 0)
            take = min(nu, end - first) - u0
            if take > 0:
                k0 = spans[s][0] + u0 * unit
                ranges.setdefault((s, grp), []).append((k0, min(k0 + take * unit, spans[s][2])))
                if take != nu:
                    parts.setdefault((s, grp), []).append(2 * block + (0 if u0 else 1))
            lo += cost[s]
            grp += 1
    return spans, ranges, parts, cost, chunk


@pytest.mark.parametrize("seed", range(8))
def test_runs_cover_every_position_once(seed):
    r = random.Random(seed)
    for _ in range(150):
        page = r.choice([12, 13, 16, 24, 40, 64])
        cap = page * r.randint(1, 300)
        unit = 512 if cap <= 512 else 128
        groups, n = r.randint(1, 5), r.randint(1, 12)
        lens = [r.choice([0, 1, r.randint(0, cap), cap, -1, cap + 5]) for _ in range(n)]
        window = r.choice([0, 0, 1, 31, 32, 33, 100, 1000])
        grid = min(r.choice([1, 2, 7, 64, 1000]), n * groups * (-(-slots(cap, page) // unit) + PAIR))
        spans, ranges, parts, cost, chunk = runs(lens, cap, window, page, groups, grid, unit)
        used = [slot for p in parts.values() for slot in p]
        assert len(used) == len(set(used)), "two partial sums in one place"
        before = 0
        for s in range(n):
            for g in range(groups):
                base, first, end, _ = spans[s]
                got = [k for a, b in ranges[(s, g)] for k in range(max(a, first), b)]
                assert got == list(range(first, end))
                # the join's view
                lo = before * groups + g * cost[s] + PAIR
                hi = lo + cost[s] - PAIR
                b0, b1 = lo // chunk, (hi - 1) // chunk
                want = [] if b0 == b1 else [2 * b + (1 if b == b0 else 0) for b in range(b0, b1 + 1)]
                assert parts.get((s, g), []) == want
            before += cost[s]


def test_division_by_page_size():
    """i / n as (i * ceil(2^(31+s) / n)) >> (31+s), s = ceil(log2 n), for every i below 2^31."""
    r = random.Random(1)
    top = (1 << 31) - 1
    for n in list(range(1, 600)) + [r.randrange(1, 1 << 20) for _ in range(1000)]:
        s = (n - 1).bit_length()
        mul = -(-(1 << (31 + s)) // n)
        assert mul < 1 << 32
        for i in [0, 1, n - 1, n, n + 1, top, top // n * n, top // n * n - 1] + [r.randrange(1 << 31) for _ in range(10)]:
            if 0 <= i <= top:
                assert (i * mul) >> (31 + s) == i // n, (i, n)


def test_argument_records_match_the_header(tmp_path):
    records = {"bb_paged_seqs": _lib.PAGED_SEQS, "bb_paged_tokens": _lib.PAGED_TOKENS,
               "bb_paged_query": _lib.PAGED_QUERY}
    last = {"bb_paged_seqs": "lens", "bb_paged_tokens": "seq_start", "bb_paged_query": "workspace_bytes"}
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(void) {\n%s return 0; }\n' % (
        _lib.HEADER, "".join(f'  printf("{n} %zu %zu\\n", sizeof({n}), offsetof({n}, {f}));\n' for n, f in last.items())))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, size, off = line.split()
        assert records[name].size == int(size)
        assert struct.calcsize(records[name].format[:-1]) <= int(off) == int(size) - 8


class NoGpu:
    """A context that no call may reach."""
    handle, device = None, 0


class Plan:
    handle = None


class Pool:
    handle, n_kv_heads, head_dim = None, 2, 64


def test_python_checks():
    plan = Plan
    x, pos = np.zeros((3, 2, 64), np.float32), np.zeros(3, np.int32)
    for args in ((x[0], pos), (x.astype(np.float64), pos), (x, pos[:2]), (x, pos.astype(np.int64)), (x[..., ::2], pos),
                 (x.astype(np.int32), pos), (x, pos, x.astype(np.float16)), (x, pos, x[:2]), (x[::-1], pos)):
        with pytest.raises(ValueError):
            kernels.rope(NoGpu, plan, *args)
    with pytest.raises(ValueError):
        kernels.rope(NoGpu, plan, x, torch.zeros(2, dtype=torch.int32))
    table, lens = np.zeros((3, 2), np.int32), np.ones(3, np.int32)
    closed = Plan
    for kw in (dict(v=x[:2]), dict(lens=lens[:2]), dict(table=table.astype(np.int64)), dict(table=table[:, ::2][:, :1].T),
               dict(q_out=x), dict(q=x[:2]), dict(rope=closed), dict(pos=pos[:2]), dict(seq_start=lens),
               dict(k_norm=np.ones(32, np.float32)), dict(q=x, q_norm=np.ones(64, np.float16)), dict(k=x[:, ::2])):
        a = dict(table=table, lens=lens, k=x, v=x) | kw
        with pytest.raises(ValueError):
            kernels.paged_append(NoGpu, Pool, a.pop("table"), a.pop("lens"), a.pop("k"), a.pop("v"), **a)
    q = np.zeros((3, 4, 64), np.float32)
    for kw in (dict(out=q[:2]), dict(out=q.astype(np.float16)), dict(q=q[:, :, :32]), dict(scale=0.0), dict(window=-1),
               dict(lse=np.zeros((3, 2), np.float32)), dict(workspace=np.zeros(1 << 20, np.uint8)),
               dict(workspace=torch.zeros(1 << 20)), dict(lens=lens[:1])):
        a = dict(lens=lens, q=q, out=q.copy()) | kw
        with pytest.raises(ValueError):
            kernels.paged_attention(NoGpu, Pool, table, a.pop("lens"), a.pop("q"), a.pop("out"), **a)
