"""What a call of prompt attention over host arrays has to have, and what it need not."""
import numpy as np
import pytest

from bebelm_amd import _lib, kernels
from bebelm_amd.model import F32
from test_gpu_paged_prompt import Pool, randn, refused, run

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
