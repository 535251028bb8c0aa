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


def check(c, got, **mask):
    want, bound = attend(c, **mask)
    n = sum(c["new"])
    assert bool(got[:n].isfinite().all())
    assert bool(((got[:n].double() - want[:n]).abs() <= bound[:n]).all())


@pytest.mark.parametrize("new", [[1, 1], [3, 1], [70, 40]])
@pytest.mark.parametrize("storage", ["16bit", "int8"])
def test_every_replay_is_the_attention_of_what_was_written(new, storage):
    """One captured step (append, attention) replayed as the sequences grow by the same numbers of tokens: each replay
    against 64 bits over everything that the replays before it wrote."""
    hq, hkv, dim, page, steps = 8, 2, 64, 16, 5
    width = -(-max(new) * steps // page)
    cache = tb.PagedKVCache.empty(2 * width + 3, page, hkv, dim, F16, DEV, storage=storage)
    table = torch.randperm(2 * width + 3, device=DEV)[:2 * width].to(torch.int32).view(2, width)
    cu, lens = torch.tensor([0, new[0], sum(new)], **I32), torch.tensor(new, **I32)
    q, k, v = (torch.randn(sum(new), h, dim, device=DEV).half() for h in (hq, hkv, hkv))

    def step():
        cache.append(k, v, table, lens, cu)
        return tb.run_paged_attn(q, cache, table, lens, cu, max_seqlen_q=max(new))

    step()
    torch.cuda.synchronize(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    kw = dict(tensor_layout="HND")
    if storage == "int8":
        kw.update(k_scale=cache.k_scale, v_scale=cache.v_scale)
    for i in range(steps):
        lens.copy_(torch.tensor([n * (i + 1) for n in new], **I32))
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize(DEV)
        assert tb.device_status(DEV) == 0
        check(dict(k=cache.k, v=cache.v, kw=kw, table=table, new=new, lens_host=lens.tolist(), q=q, total=sum(new), dtype=F16,
                   heads=(hq, hkv, dim), page=page), o)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_whole_prompts_element_by_element_beside_the_packed_call(dtype, dim):
    """Prompts with nothing before them are run_flash_attn_varlen's causal case. Both results are within their bound of
    the same value: attend()'s for the cache's; half as much again for the packed call, whose exponential is off by up to
    2^-13, in a weight and in their sum: 2^-12 of sum w |v|, at most half of u = 2^-11 (2^-8) of it."""
    new = [300, 65, 1, 128]
    c = make_case(DEV, new=new, past=[0] * 4, hq=8, hkv=2, dim=dim, page=32, dtype=dtype, seed=21)
    cache = tb.PagedKVCache(c["k"], c["v"], **c["kw"])
    k, v = (torch.randn(sum(new), 2, dim, device=DEV).to(dtype) for _ in range(2))
    cache.append(k, v, c["table"], c["lens"], c["cu"])
    a = tb.run_paged_attn(c["q"], cache, c["table"], c["lens"], c["cu"], max_seqlen_q=300)
    b = tb.run_flash_attn_varlen(c["q"], k, v, c["cu"], c["cu"], causal=True)
    want, bound = attend(c)
    assert bool(((a.double() - want).abs() <= bound).all())
    assert bool(((a.double() - b.double()).abs() <= 2.5 * bound).all())


@pytest.mark.parametrize("bound", ["largest", "none"])
@pytest.mark.parametrize("storage", ["16bit", "int8"])
@pytest.mark.parametrize("chunks", [[150, 90], [40, 200, 33], [300]])
def test_single_tokens_beside_several_chunks(chunks, storage, bound):
    new = [1] * 20 + chunks + [1] * 9 + [2, 0]
    past = [(i * 211) % 800 for i in range(len(new))]
    c = make_case(DEV, new=new, past=past, hq=8, hkv=2, dim=128, page=16, dtype=BF16, storage=storage, mean=storage == "int8", seed=22)
    cache = tb.PagedKVCache(c["k"], c["v"], **c["kw"])
    o = tb.run_paged_attn(c["q"], cache, c["table"], c["lens"], c["cu"], **(dict(max_seqlen_q=c["max_new"]) if bound == "largest" else {}))
    check(c, o)
