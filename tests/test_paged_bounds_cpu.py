"""CPU: the bound max_seqlen_q of paged attention may lie far above the number of tokens."""
import ctypes

import pytest

from tribench_b200 import _native as N


@pytest.mark.parametrize("storage", [N.SAGE_CACHE_16BIT, N.SAGE_CACHE_INT8])
@pytest.mark.parametrize("batch,total", [(2, 1000), (1, 1), (64, 64 + 511), (16, 16)])
@pytest.mark.parametrize("heads", [2, 8, 16])
def test_a_bound_above_the_tokens_counts_as_their_number(storage, batch, total, heads):
    c = N.PagedCacheStruct(page_size=16, heads_kv=2, head_dim=64, num_pages=4, dtype=N.SAGE_DTYPE_F16, storage=storage)

    def size(bound):
        return N.load().sage_paged_workspace_bytes(ctypes.byref(c), heads, batch, total, bound, 64)

    want = size(total)
    assert want > 0
    for bound in (total + 1, 1 << 31, 1 << 62, (1 << 63) - 1):
        assert size(bound) == want
