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
