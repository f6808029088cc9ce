"""Scores of attention over a paged cache where their size goes past the usual, against the formulas of
tests/test_gpu_paged_prompt.py in 64 bits. Caps far above the scores they shape: the tolerances there hold (a capped score is
off by 12 steps of itself, however large the cap). Scores as large as f32 holds."""
import math

import numpy as np
import pytest
import torch

from bebelm_amd import kernels
from bebelm_amd.model import BF16, F16, F32, KV4
from test_gpu_paged_prompt import (INF, TINY, TYPES, U, Pool, check, close, done, gen, half_step, held, i32, on_gpu, randn, run,
                                   slopes_of)

pytestmark = pytest.mark.gpu


# ---- caps ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cap", [1.0, 50.0, 64.0, 65.0, 1e3, 1e4, 1e5, 1e6, 1e9])
@pytest.mark.parametrize("dt,ct", [(F16, F16), (BF16, BF16), (BF16, F16), (F16, KV4), (F32, F32), (F32, BF16)])
def test_caps_far_above_the_scores(gpu_ctx, cap, dt, ct):
    """Scores of a few units and of hundreds under caps of every size, tokens in tiles and one each."""
    print("cap", cap, dt, ct, flush=True)
    for hd, bring, before in ((64, [40, 3], [30, 200]), (128, [90, 17], [0, 100])):
        pool = Pool(gpu_ctx, 110, [a + b for a, b in zip(before, bring)], ct, 16, 2, hd)
        q = randn(111, (sum(bring), 4, hd), dt)
        for scale in (0.125, 4.0):
            check(gpu_ctx, pool, q, dt, bring, scale=scale, cap=cap, what=f"hd {hd} scale {scale}")
        check(gpu_ctx, pool, q, dt, bring, cap=cap, slopes=slopes_of(4), window=50, prefix=[3, 0])
        check(gpu_ctx, pool, q[:2], dt, [1, 1], scale=4.0, cap=cap, single=True)


@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1e-30, 1e25, 1e30, 1e36, 2e38, 3.4e38])
@pytest.mark.parametrize("dt,ct", [(F16, F16), (BF16, BF16), (F32, F16), (F16, KV4), (F32, F32), (F32, BF16), (BF16, F16)])
def test_caps_at_the_ends_of_the_range(gpu_ctx, cap, dt, ct):
    """Ordinary scores, and queries of small elements: under the largest caps as without one, under the smallest all equal."""
    print("cap", cap, dt, ct, flush=True)
    for hd, bring, before in ((64, [40, 3], [30, 200]), (128, [90, 17], [0, 100])):
        pool = Pool(gpu_ctx, 112, [a + b for a, b in zip(before, bring)], ct, 16, 2, hd)
        q = randn(113, (sum(bring), 4, hd), dt)
        q[:, 1] *= 2.0 ** -10
        q[3] = 0
        for kw in (dict(), dict(scale=2.0, window=33)):
            check(gpu_ctx, pool, q, dt, bring, cap=cap, what=f"hd {hd} {kw}", **kw)
            check(gpu_ctx, pool, q[2:4], dt, [1, 1], cap=cap, single=True, what=f"single hd {hd} {kw}", **kw)


# ---- large scores ----------------------------------------------------------------------------------------
# Scores that are products of one element each, exact in f32: a query's, times a key's of a few levels. So scores are
# equal, and their weights too, or a quarter of the largest apart: from 1000 on the lower one's weight is 0 in f32. What is
# left are the roundings of the sums and of 16-bit weights, and of lse its own: of the score's product with scale·log2(e), of that
# factor, of the sum with the weights' log, of the product with log(2), of that: 5 steps.
LEVELS = [1.0, 0.75, 0.5, 0.25, -0.25, -1.0]


def levels(ctx, seed, lens, ct, kv, hd, order):
    """A pool whose keys have one element each, of LEVELS (as the pool holds them), in the given order along a sequence."""
    pool = Pool(ctx, seed, lens, ct, 16, kv, hd)
    total, g = sum(lens), gen(seed + 5)
    pick = torch.randint(0, len(LEVELS), (total, kv), generator=g)
    if order != "any":
        at = 0
        for n in lens:
            pick[at:at + n] = pick[at:at + n].sort(0, descending=order == "rising")[0]
            at += n
    k = torch.zeros(total, kv, hd)
    k[:, :, 5] = torch.tensor(LEVELS)[pick]
    v = torch.randn(total, kv, hd, generator=g)
    start = [0] + np.cumsum(lens).tolist()
    table, ln, kd, vd, st = on_gpu(pool.table, pool.lens, k, v, i32(start))
    kernels.paged_append(ctx, pool.kv, table, ln, kd, vd, seq_start=st)
    done(ctx)
    kept = [held(x) if ct == KV4 else x.to(TYPES[ct]).double() for x in (k, v)]
    return pool, [tuple(x[start[s]:start[s + 1]] for x in kept) for s in range(len(lens))]


def check_levels(ctx, pool, history, q, dt, bring, scale, single=False, window=0, **kw):
    scale = float(np.float32(scale))
    start = [0] + np.cumsum(bring).tolist()
    out, lse = run(ctx, pool, q, None if single else start, scale=scale, window=window, **kw)
    for s, n in enumerate(bring):
        length, rows = pool.lens_list[s], slice(start[s], start[s + 1])
        k, v = history[s]
        i, j = torch.arange(length - n, length)[:, None, None], torch.arange(length)
        # (by differences from the largest: 64 bits do not hold a large score's sum with a weight's log)
        x = (q[rows].double() @ k[:, 0].T) * scale
        x = x.masked_fill(~((j <= i) & ((i - j < window) if window else torch.ones(1, dtype=torch.bool))), -INF)
        most = x.amax(-1, keepdim=True)
        p = torch.exp(x - most)
        want, wl = p @ v[:, 0] / p.sum(-1, keepdim=True), most[..., 0] + torch.log(p.sum(-1))
        # ordinary scores (a head of small queries) are off by 8 steps of the largest
        top = x.masked_fill(torch.isinf(x), 0.0).abs().amax(-1)
        d = torch.where(top < 1000, 8 * U * top, 0.0)
        # f16 parts of a query are multiples of its largest element's power of two, which is put at 2^13: an element is off by
        # half of f16's smallest step, 2^-25, or 2^-38 of that (where the scored element is the largest it is exact)
        if pool.ct in (F16, KV4):
            most_q = q[rows].double().abs().amax(-1)
            d = torch.where(q[rows][..., 5].double().abs() < most_q, d + 2.0 ** -38 * most_q * abs(scale) * k.abs().amax(), d)
        # (every weight is off by up to: sums, the weight's own rounding)
        w16 = {BF16: 2.0 ** -8 if pool.ct == BF16 else 2.0 ** -11, F16: 2.0 ** -11, F32: 0.0}[dt]
        tol = 2 * d + 2 * (8 * math.sqrt(length) + 16) * U + w16
        tol = (tol[..., None] + length * 2.0 ** -33) * v.abs().amax()
        what = f"scale {scale:g} window {window} single {single} sequence {s}"
        close(out[rows], want, tol * (1 + half_step(dt)) + half_step(dt) * want.abs() + TINY[dt], f"out {what}")
        close(lse[rows], wl, 5 * U * wl.abs() + d + (8 * math.sqrt(length) + 16) * U, f"lse {what}")


@pytest.mark.parametrize("order", ["any", "rising", "falling"])
@pytest.mark.parametrize("dt,ct", [(F16, F16), (BF16, BF16), (F32, F16), (F16, KV4), (F32, KV4), (F32, F32), (F32, BF16),
                                   (BF16, F16)])
def test_large_scores(gpu_ctx, order, dt, ct):
    """Tiles of 128 rows and of few, parts that are joined; with a bias of 0 (scores are then made before the maximum
    is taken)."""
    print("large", order, dt, ct, flush=True)
    for hd, heads in ((64, 4), (128, 2), (256, 2)):
        pool, history = levels(gpu_ctx, 120, [140, 33], ct, 1, hd, order)
        few, behind = levels(gpu_ctx, 130, [1400], ct, 1, hd, order)
        q = torch.zeros(160, heads, hd)
        q[:, :, 5] = 8.0
        if dt != F16:
            q[1::2, 1, 5] = 2.0 ** -40     # a row of other size in the same tile
        q[:, :, 6:] = 1.0                  # (times keys of 0)
        q = q.to(TYPES[dt])
        for scale in (1e4, 3e6, 5e6, 1.1e7, 1.7e7, 3e7, 1e8, 1e10, -1e10, 1e20, 1e30, 5e36):
            for kw in (dict(), dict(window=20), dict(slopes=torch.zeros(heads))):
                check_levels(gpu_ctx, pool, history, q, dt, [130, 30], scale, **kw)
            for n in (2, 9, 17):
                check_levels(gpu_ctx, few, behind, q[:n], dt, [n], scale)


@pytest.mark.parametrize("order", ["any", "rising", "falling"])
@pytest.mark.parametrize("dt,ct", [(F16, F16), (BF16, BF16), (F16, KV4), (F32, KV4), (F32, F32), (F32, BF16)])
def test_large_scores_of_single_tokens(gpu_ctx, order, dt, ct):
    """The same, one token each."""
    print("large, single", order, dt, ct, flush=True)
    for hd, heads in ((64, 4), (128, 2), (256, 2)):
        pool, history = levels(gpu_ctx, 140, [140, 33, 1400], ct, 1, hd, order)
        q = torch.zeros(3, heads, hd)
        q[:, :, 5] = 8.0 * 2.0 ** -torch.arange(heads)   # (heads that pass 2^16 at different positions)
        q = q.to(TYPES[dt])
        for scale in (1e4, 2e4, 3e6, 5e6, 1.1e7, 1.7e7, 3e7, 1e8, 1e10, -1e10, 1e20, 1e30, 5e36):
            for kw in (dict(), dict(window=20), dict(slopes=torch.zeros(heads))):
                check_levels(gpu_ctx, pool, history, q, dt, [1, 1, 1], scale, single=True, **kw)
