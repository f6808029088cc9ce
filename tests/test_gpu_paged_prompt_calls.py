"""What a call of prompt attention over host arrays has to have, and what it need not."""
import numpy as np
import pytest
import torch

from bebelm_amd import _lib, kernels
from bebelm_amd.model import F32
from test_gpu_paged_prompt import Pool, done, randn, refused, run

pytestmark = pytest.mark.gpu


def test_pages_that_no_token_reads_need_not_be_there(gpu_ctx):
    """A sequence that brings no tokens needs no pages, whatever its prefix; one that does, those of its prefix."""
    pool = Pool(gpu_ctx, 150, [40, 50, 0], F32, 16, 2, 64)
    q, start = randn(151, (12, 4, 64), F32), [0, 12, 12, 12]
    want, wl = run(gpu_ctx, pool, q, start, window=5)
    gone = pool.table.clone()
    gone[1] = -1
    out, lse = np.full((12, 4, 64), 7.0, np.float32), np.full((12, 4), 7.0, np.float32)

    def call(prefix, table=gone):
        return kernels.paged_prompt_attention(gpu_ctx, pool.kv, table.numpy(), pool.lens.numpy(), q.numpy(), out,
                                              seq_start=np.array(start, np.int32), window=5,
                                              prefix=np.array(prefix, np.int32), lse=lse)

    for prefix in ([0, 0, 0], [0, 20, 0], [0, 1 << 30, 9]):
        call(prefix)
        assert np.array_equal(out, want.numpy()) and np.array_equal(lse, wl.numpy())
    refused(_lib.BB_ERR_RANGE, lambda: call([0, -1, 0]))
    gone[0, 0] = 1 << 30
    call([0, 20, 0])
    refused(_lib.BB_ERR_RANGE, lambda: call([1, 20, 0]))


def test_scales_that_base_2_does_not_hold_are_refused(gpu_ctx):
    """Scores are exponents of 2: a scale whose product with log2(e) is infinite would make NaN of a score of 0."""
    pool = Pool(gpu_ctx, 152, [40, 50], F32, 16, 2, 64)
    q = torch.zeros(2, 4, 64, device="cuda")
    out, table, lens = torch.full_like(q, 7.0), pool.table.cuda(), pool.lens.cuda()
    for scale in (2.0 ** 127, -(2.0 ** 127), 3.4e38, float("inf"), float("nan")):
        refused(_lib.BB_ERR_ARG, lambda: kernels.paged_prompt_attention(gpu_ctx, pool.kv, table, lens, q, out, scale=scale))
        refused(_lib.BB_ERR_ARG, lambda: kernels.paged_attention(gpu_ctx, pool.kv, table, lens, q, out, scale=scale))
    assert bool((out == 7.0).all())
    for call in (kernels.paged_prompt_attention, kernels.paged_attention):   # (below it: a mean of the values)
        call(gpu_ctx, pool.kv, table, lens, q, out, scale=1.7e38)
        done(gpu_ctx)
        for s in range(2):
            v = pool.history(s)[1].mean(0).repeat_interleave(2, 0)
            # (a sum of 50 values below 4 and its quotient: 8·sqrt(50) + 8 half steps)
            assert torch.allclose(out[s].cpu().double(), v, rtol=0, atol=64 * 2.0 ** -24 * 4)
        out.fill_(7.0)
