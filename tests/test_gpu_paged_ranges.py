"""GPU: attention over an INT8 cache whose rows differ widely in size, against the 64-bit implementation and bound of
paged_ref.py. The bound knows of no key but by its weight: a value row weighs in 16 bits relative to the largest weight
times scale that its query has, whatever the scales of keys that this query does not see or hardly attends to."""
import pytest
import torch

import tribench_b200 as tb
from paged_ref import attend, make_case

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16 = torch.float16, torch.bfloat16


def cache_of(c):
    return tb.PagedKVCache(c["k"], c["v"], **c["kw"])


def run(c, **mask):
    o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=c["max_new"], **mask)
    assert tb.device_status(DEV) == 0
    return o


def worst(c, got, rows=None, **mask):
    """The largest error in units of its bound, over packed rows [0, rows)."""
    want, bound = attend(c, **mask)
    rows = sum(c["new"]) if rows is None else rows
    got, want, bound = got[:rows].double(), want[:rows], bound[:rows]
    assert bool(got.isfinite().all())
    return ((got - want).abs() / bound.clamp(min=1e-300)).max().item()


def place(c, b, pos):
    """(page, row) of a position of sequence b."""
    return int(c["table"][b, pos // c["page"]]), pos % c["page"]


def each_scale(c, name, factor):
    """Multiplies the scale of every position p of sequence 0 by factor[p]."""
    p = torch.arange(c["lens_host"][0], device=DEV)
    c["kw"][name][c["table"][0].long()[p // c["page"]], :, p % c["page"]] *= factor[:, None]


@pytest.mark.parametrize("n", [4, 100])
@pytest.mark.parametrize("past", [20, 150])
@pytest.mark.parametrize("dtype,top", [(F16, 65504.0), (BF16, 1e6), (BF16, 3e38)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_later_tokens_value_leaves_earlier_rows_alone(n, past, dtype, top, dim):
    """The last token's key and value are far larger than all others: the tokens before it do not see them."""
    c = make_case(DEV, new=[n], past=[past], hq=4, hkv=2, dim=dim, page=16, dtype=dtype, storage="int8", seed=15)
    pg, row = place(c, 0, past + n - 1)
    for x in ("k_scale", "v_scale"):
        c["kw"][x][pg, :, row] = top / 127
    assert worst(c, run(c), rows=n - 1) <= 1


@pytest.mark.parametrize("n", [1, 3, 8, 100])
@pytest.mark.parametrize("log2_weight", [-30, -90])
@pytest.mark.parametrize("log2_size", [8, 16, 26, 60, 120])
def test_a_large_value_row_of_little_weight(n, log2_weight, log2_size):
    """One key of the first tile holds values 2^r larger than the rest and next to no weight. Splits along the keys
    (few sequences, many keys) put it into another part than most keys."""
    for past in (100, 6000):
        c = make_case(DEV, new=[n], past=[past], hq=4, hkv=2, dim=128, page=16, dtype=BF16, storage="int8", seed=3)
        c["q"][..., 0] = 8.0
        pg, row = place(c, 0, 3)
        # its score is about log2_weight ln 2 below the others': 8 x dim^-1/2
        c["k"][pg, :, row] = 0
        c["k"][pg, :, row, 0] = -127
        c["kw"]["k_scale"][pg, :, row] = -log2_weight * 0.6931 * 128 ** 0.5 / 8 / 127
        c["kw"]["v_scale"][pg, :, row] = 0.01 * 2.0 ** log2_size
        assert worst(c, run(c)) <= 1


@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("shape", ["up", "down", "there_and_back", "random", "steps"])
@pytest.mark.parametrize("span", [7, 20, 60])
def test_scales_that_change_along_the_sequence(n, shape, span):
    """Value scales over 2^span, rising, falling, both, at random per token, and in steps of tiles."""
    past = 1500
    c = make_case(DEV, new=[n], past=[past], hq=4, hkv=2, dim=64, page=32, dtype=BF16, storage="int8", seed=4)
    p = torch.arange(past + n, device=DEV).double() / (past + n)
    g = torch.Generator(device=DEV).manual_seed(8)
    e = {"up": p, "down": 1 - p, "there_and_back": 1 - (2 * p - 1).abs(), "steps": torch.floor(p * 5) % 2,
         "random": torch.rand(past + n, generator=g, device=DEV).double()}[shape]
    each_scale(c, "v_scale", (2.0 ** (span * (e - 0.5))).float())
    assert worst(c, run(c)) <= 1
    assert worst(c, run(c, window=300, sinks=3), window=300, sinks=3) <= 1


@pytest.mark.parametrize("n", [1, 6, 90])
def test_a_sink_with_small_values(n):
    """A first key that takes nearly all weight and whose values are tiny or zero: what is left comes from the others."""
    for scale in (1e-6, 0.0):
        c = make_case(DEV, new=[n], past=[700], hq=4, hkv=2, dim=128, page=16, dtype=F16, storage="int8", seed=5)
        c["q"][..., 0] = 8.0
        pg, row = place(c, 0, 0)
        c["k"][pg, :, row] = 0
        c["k"][pg, :, row, 0] = 127
        c["kw"]["k_scale"][pg, :, row] = 15 / 127
        c["kw"]["v_scale"][pg, :, row] = scale
        assert worst(c, run(c)) <= 1


@pytest.mark.parametrize("n", [1, 90])
def test_zero_and_huge_values(n):
    """Value rows that are all zero give zero; rows near the type's largest come back as such; a mixture too."""
    c = make_case(DEV, new=[n], past=[300], hq=4, hkv=2, dim=128, page=16, dtype=BF16, storage="int8", seed=6)
    s = c["kw"]["v_scale"]
    s.nan_to_num_(nan=0.0).zero_()
    assert bool((run(c) == 0).all())
    s.fill_(2.0 ** 120)
    assert worst(c, run(c)) <= 1
    s[:, :, ::2] = 2.0 ** -100
    s[:, :, 1::4] = 0.0
    assert worst(c, run(c)) <= 1


@pytest.mark.parametrize("n", [1, 30])
def test_negative_scales(n):
    """code * scale holds for scales of either sign."""
    c = make_case(DEV, new=[n], past=[300], hq=4, hkv=2, dim=64, page=16, dtype=F16, storage="int8", seed=9)
    for x in ("k_scale", "v_scale"):
        c["kw"][x] *= torch.where(torch.rand_like(c["kw"][x]) < 0.5, -1.0, 1.0)
    # the bound asks for sizes: fold the signs into the codes
    plain = dict(c, k=c["k"] * c["kw"]["k_scale"].sign().nan_to_num(1)[..., None].to(torch.int8),
                 v=c["v"] * c["kw"]["v_scale"].sign().nan_to_num(1)[..., None].to(torch.int8),
                 kw=dict(c["kw"], k_scale=c["kw"]["k_scale"].abs(), v_scale=c["kw"]["v_scale"].abs()))
    assert worst(plain, run(c)) <= 1


@pytest.mark.parametrize("n", [1, 60])
def test_wide_scales_beside_plain_sequences(n):
    """Sequences of one call, one with wide scales, one without: each as if alone, and the same bits twice."""
    c = make_case(DEV, new=[n, n, n], past=[900, 40, 5000], hq=8, hkv=2, dim=128, page=16, dtype=BF16, storage="int8", seed=10)
    g = torch.Generator(device=DEV).manual_seed(2)
    each_scale(c, "v_scale", 2.0 ** (40 * torch.rand(900 + n, generator=g, device=DEV) - 20))
    o = run(c)
    assert worst(c, o) <= 1
    assert torch.equal(o, run(c))


@pytest.mark.parametrize("n", [1, 4, 100])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_that_is_not_finite(n, bad, dim):
    """A key row with an infinity or a NaN is held as NaN: queries that see it get NaN, the others do not notice."""
    for at in (3, 40, 41 + n - 1):
        c = make_case(DEV, new=[n], past=[41], hq=4, hkv=2, dim=dim, page=16, dtype=F16, storage="int8", seed=11)
        cache = cache_of(c)
        one = torch.randn(1, 2, dim, device=DEV).half()
        k = one.clone()
        k[0, :, 5] = bad
        i32 = dict(dtype=torch.int32, device=DEV)
        cache.append(k, one, c["table"], torch.tensor([at + 1], **i32))
        assert bool(cache.gather(c["table"], torch.tensor([at + 1], **i32))[0].isnan().all())
        o = run(c)
        unseen = max(at - 41, 0)  # rows before the key
        assert bool(o[unseen:].isnan().all())
        # to the bound's arithmetic the key does not exist for rows before it
        c["kw"]["k_scale"].nan_to_num_(nan=0.0, posinf=0.0)
        if unseen:
            assert worst(c, o, rows=unseen) <= 1


@pytest.mark.parametrize("n", [1, 4, 100])
@pytest.mark.parametrize("log2", [-110, -60, 60, 100, 118])
def test_queries_of_any_size(n, log2):
    """Queries far from 1 with keys that make up for it: scores are as usual."""
    c = make_case(DEV, new=[n], past=[200], hq=4, hkv=2, dim=128, page=16, dtype=BF16, storage="int8", seed=12)
    c["q"] = (c["q"].double() * 2.0 ** log2).to(BF16)
    c["kw"]["k_scale"] *= 2.0 ** -log2
    assert worst(c, run(c)) <= 1


@pytest.mark.parametrize("n", [40, 130])
@pytest.mark.parametrize("span", [10.0, 10.9, 11.1, 12.0])
@pytest.mark.parametrize("drift", [0, 25, 31, 45, -28, -33, -60])
def test_where_the_chunk_kernel_changes_its_units(n, span, drift):
    """Scales spread over 2^span within each tile, and drifting by 2^drift along the sequence: about what one unit per
    tile takes (2^11), and how far it moves within a segment (2^30)."""
    past = 1100
    c = make_case(DEV, new=[n], past=[past], hq=4, hkv=2, dim=64, page=64, dtype=BF16, storage="int8", seed=23)
    c["kw"]["v_scale"] = torch.where(c["kw"]["v_scale"].isnan(), c["kw"]["v_scale"], 1.0)
    g = torch.Generator(device=DEV).manual_seed(3)
    e = span * torch.rand(past + n, generator=g, device=DEV) + drift * torch.arange(past + n, device=DEV) / (past + n)
    each_scale(c, "v_scale", 2.0 ** (e - 8))
    assert worst(c, run(c)) <= 1
    assert worst(c, run(c, window=500, sinks=130), window=500, sinks=130) <= 1
