"""Scores of attention over a paged cache where their size goes past the usual: caps far above the scores they shape, against
the formulas of tests/test_gpu_paged_prompt.py in 64 bits, whose tolerances hold (a capped score is off by 12 steps of
itself, however large the cap)."""
import pytest
import torch

from bebelm_amd.model import BF16, F16, F32, KV4
from test_gpu_paged_prompt import Pool, check, randn, slopes_of

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
