"""GPU: the paged cache in use: what its object allows, replays of captured calls against the 64-bit implementation, and
the packed attention call on the same prompt."""
import pytest
import torch

import tribench_b200 as tb
from paged_ref import attend, make_case

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16 = torch.float16, torch.bfloat16
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("storage", ["16bit", "int8"])
def test_tensors_of_a_cache_cannot_be_exchanged(storage):
    """The calls hold the addresses of construction: another tensor in their place would leave them with freed memory."""
    cache = tb.PagedKVCache.empty(4, 16, 2, 64, F16, DEV, storage=storage)
    for name in ("k", "v", "k_scale", "v_scale", "k_mean", "dtype", "num_pages", "heads_kv", "page_size", "head_dim"):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(cache, name, getattr(cache, name))
    cache.k.zero_()
    cache.note = 1  # anything else may be attached
