"""GPU: the paged key/value cache (append, gather) and attention over it, against a plain implementation in 64
bits (paged_ref.py, which derives the attention tolerance)."""
import pytest
import torch

import tribench_b200 as tb
import tribench_b200._native  # noqa: F401
from paged_ref import attend, held, make_case

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16 = torch.float16, torch.bfloat16


def cache_of(c):
    return tb.PagedKVCache(c["k"], c["v"], **c["kw"])


# ------------------------------------------------------------------ write and read back
def _codes(x):
    """Codes and scales of rows of x (fp32) as the definition gives them; `sure`: not within fp32 error of a tie."""
    a = x.abs().amax(-1, keepdim=True)
    exact = torch.where(a > 0, x.double() * 127 / a.double(), torch.zeros_like(x, dtype=torch.float64))
    # 127 x and the quotient each round to fp32 (2^-24 relative, |quotient| <= 127)
    sure = ((exact - exact.floor()) - 0.5).abs() > 127 * 2.0 ** -23
    return torch.round(exact), (a.double() / 127).float()[..., 0], sure  # fp32 tensors divide by a number inexactly


@pytest.mark.parametrize("new,past,hkv,dim,page,dtype,storage,layout,mean", [
    ([1], [0], 1, 64, 16, F16, "16bit", "HND", False),
    ([1, 1, 1], [15, 16, 40], 8, 128, 16, BF16, "16bit", "NHD", False),
    ([5, 0, 70, 1], [11, 3, 0, 63], 3, 128, 32, F16, "int8", "HND", False),
    ([33, 129], [100, 0], 2, 64, 64, BF16, "int8", "NHD", False),
    ([200, 0, 0, 3], [0, 0, 9, 1000], 5, 128, 1024, F16, "int8", "HND", True),
    ([17, 31], [1, 2], 16, 64, 16, BF16, "int8", "HND", True),
    ([1] * 100, [i * 7 % 90 for i in range(100)], 2, 64, 16, F16, "16bit", "HND", False),
])
def test_append_then_gather(new, past, hkv, dim, page, dtype, storage, layout, mean):
    c = make_case(DEV, new=new, past=past, hq=hkv, hkv=hkv, dim=dim, page=page, dtype=dtype, storage=storage, layout=layout,
                  mean=mean, seed=dim + page, spare_rows=2)
    cache = cache_of(c)
    g = torch.Generator(device=DEV).manual_seed(5)
    k = (torch.randn(c["total"], hkv, dim, generator=g, device=DEV) * 3 + 1).to(dtype)
    v = torch.randn(c["total"], hkv, dim, generator=g, device=DEV).to(dtype)
    v[0] = 0  # a row of zeros: scale 0, codes 0
    state = {n: t.clone() for n, t in (("k", c["k"]), ("v", c["v"]), ("ks", c["kw"].get("k_scale")), ("vs", c["kw"].get("v_scale")))
             if t is not None}
    cache.append(k, v, c["table"], c["lens"], c["cu"])
    # what is expected, by plain indexing into copies
    n = sum(new)
    pg, row = [], []
    for b, m in enumerate(new):
        pos = torch.arange(c["lens_host"][b] - m, c["lens_host"][b], device=DEV)
        pg.append(c["table"][b].long()[pos // page])
        row.append(pos % page)
    pg, row = torch.cat(pg), torch.cat(row)
    hnd = (lambda t: t.transpose(1, 2)) if layout == "NHD" else (lambda t: t)
    back = []
    for name, x, off in (("k", k[:n], c["kw"].get("k_mean")), ("v", v[:n], None)):
        want = hnd(state[name])
        if storage == "16bit":
            want[pg, :, row] = x
            assert torch.equal(hnd(c[name]).nan_to_num(7), want.nan_to_num(7))
            back.append(x)
            continue
        y = x.float() if off is None else x.float() - off
        code, scale, sure = _codes(y)
        got = hnd(c[name])[pg, :, row]
        if off is None:
            assert torch.equal(got.double(), code)  # 16-bit values: no quotient is near a tie it is not on
        else:
            assert torch.equal(got.double()[sure], code[sure]) and (got.double() - code).abs().max() <= 1
        scales = c["kw"][name + "_scale"]
        assert torch.equal(scales[pg, :, row], scale)
        want[pg, :, row] = got
        assert torch.equal(hnd(c[name]), want)  # and nothing else was written
        state[name + "s"][pg, :, row] = scale
        assert torch.equal(scales.nan_to_num(7), state[name + "s"].nan_to_num(7))
        z = got.float() * scale[..., None]
        back.append((z if off is None else z + off).to(dtype))
    ko, vo = (torch.full((c["total"], hkv, dim), 9.0, dtype=dtype, device=DEV) for _ in range(2))
    cache.gather(c["table"], c["lens"], c["cu"], out=(ko, vo))
    assert torch.equal(ko[:n], back[0]) and torch.equal(vo[:n], back[1])
    assert bool((ko[n:] == 9).all()) and bool((vo[n:] == 9).all())  # rows behind the last sequence
    k2, v2 = cache.gather(c["table"], c["lens"], c["cu"], total=c["total"])
    assert torch.equal(k2[:n], ko[:n]) and torch.equal(v2[:n], vo[:n])


def test_ties_round_to_even():
    # a = 127: codes are rint(x): halves go to the even code
    cache = tb.PagedKVCache.empty(1, 16, 1, 64, F16, DEV, storage="int8")
    x = torch.zeros(1, 1, 64, device=DEV)
    x[0, 0, :8] = torch.tensor([127, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -125.5])
    one = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    cache.append(x.half(), x.half(), one, one[0] + 1)
    assert cache.k[0, 0, 0, :8].tolist() == [127, 0, 2, 2, 0, -2, 126, -126]
    assert float(cache.k_scale[0, 0, 0]) == 1.0


@pytest.mark.parametrize("top", [1e-39, 1e-35, 2.0 ** -100, 1e-20, 1e20, 1e33, 3.3e38])
def test_rows_of_any_size(top):
    """Codes of bf16 rows at both ends of the type's range, subnormal ones among them: the nearest, as 64 bits say."""
    cache = tb.PagedKVCache.empty(1, 16, 1, 128, BF16, DEV, storage="int8")
    x = (torch.rand(16, 1, 128, device=DEV, dtype=torch.float64) * 2 - 1).mul_(top).to(BF16)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    lens, cu = torch.tensor([16], dtype=torch.int32, device=DEV), torch.tensor([0, 16], dtype=torch.int32, device=DEV)
    cache.append(x, x, table, lens, cu)
    y = x.double()[:, 0]
    a = y.abs().amax(-1, keepdim=True)
    want = torch.round(y * 127 / a)
    assert torch.equal(cache.k[0, 0].double(), want) and torch.equal(cache.v[0, 0].double(), want)
    # a subnormal scale keeps fewer bits: half of the least subnormal, 2^-149
    assert bool(((cache.k_scale[0, 0].double() - a[:, 0] / 127).abs() <= a[:, 0] / 127 * 2.0 ** -24 + 2.0 ** -150).all())


def test_rows_that_are_not_finite_read_back_as_nan():
    cache = tb.PagedKVCache.empty(1, 16, 1, 64, BF16, DEV, storage="int8")
    x = torch.ones(3, 1, 64, device=DEV, dtype=BF16)
    x[1, 0, 3], x[2, 0, 63] = float("inf"), float("nan")
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    lens, cu = torch.tensor([3], dtype=torch.int32, device=DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    cache.append(x, x, table, lens, cu)
    k, v = cache.gather(table, lens, cu, total=3)
    for t in (k, v):
        assert bool((t[0] == 1).all()) and bool(t[1:].isnan().all())


def test_bad_pages_and_lengths_stay_inside():
    """Page numbers outside the cache, lengths past the page table, more new tokens than held and prefix sums that
    run off the packed tensor: writes are skipped, reads give zeros, nothing else changes."""
    cache = tb.PagedKVCache.empty(4, 16, 2, 64, F16, DEV)
    cache.k.fill_(1), cache.v.fill_(2)
    x = torch.full((40, 2, 64), 5.0, dtype=F16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.tensor([[-1, 4], [2, 1 << 30], [3, -7]], **i32)
    lens = torch.tensor([20, 1000000, 2], **i32)  # the second: 32 positions fit
    cu = torch.tensor([0, 4, 14, 24], **i32)
    cache.append(x, x, table, lens, cu)
    # sequence 0: no good page. 1: positions 22 .. 31 lie on its bad page. 2: 10 new of 2 held: positions 0, 1.
    want = torch.ones(4, 2, 16, 64, dtype=F16, device=DEV)
    want[3, :, :2] = 5
    assert torch.equal(cache.k, want)
    k, v = cache.gather(table, lens, cu, total=24)
    assert bool((k[:22] == 0).all()) and bool((k[22:24] == 5).all()) and bool((v[22:24] == 5).all())
    q = torch.randn(24, 4, 64, device=DEV).half()
    for n in (1, 10):
        o = tb.run_paged_attn(q, cache, table, lens, cu, max_seqlen_q=n)
        # with a bound of 1 only each sequence's first row is its
        assert bool((o[22:24] if n == 10 else o[14:15]).isfinite().all()) and tb.device_status(DEV) == 0
    before = cache.k.clone()
    for cu in ([0, 100, 200, 300], [5, 3, -1, 2], [39, 45, 1 << 30, -(1 << 30)], [-5, 0, 3, 9]):
        cu = torch.tensor(cu, **i32)
        cache.gather(table, lens, cu, total=24)
        tb.run_paged_attn(q, cache, table, lens, cu, max_seqlen_q=7)
        cache.append(x[:24], x[:24], table, torch.zeros_like(lens), cu)  # no token has a position
    assert torch.equal(cache.k, before) and tb.device_status(DEV) == 0


# ------------------------------------------------------------------ attention
CASES = [
    # new, past, hq, hkv, dim, page, dtype, storage, options
    ([1], [0], 1, 1, 64, 16, F16, "16bit", {}),
    ([1], [0], 8, 2, 128, 16, BF16, "int8", {}),
    ([1, 1, 1, 1], [0, 62, 63, 64], 4, 4, 128, 16, F16, "16bit", {}),
    ([1, 1, 1], [127, 1000, 5], 32, 8, 128, 64, BF16, "16bit", {}),
    ([1, 1, 1], [127, 1000, 5], 32, 8, 128, 64, BF16, "int8", {"mean": True}),
    ([1, 0, 1], [30, 12, 500], 16, 1, 64, 32, F16, "int8", {}),
    ([1, 1], [3000, 41], 64, 4, 128, 128, F16, "16bit", {}),
    ([1] * 37, [(i * 131) % 700 for i in range(37)], 8, 2, 64, 16, BF16, "16bit", {}),
    ([1] * 37, [(i * 131) % 700 for i in range(37)], 5, 1, 128, 16, F16, "int8", {"layout": "NHD"}),
    ([4, 1, 3, 8], [100, 0, 1, 777], 6, 2, 64, 16, F16, "16bit", {}),
    ([4, 1, 3, 8], [100, 0, 1, 777], 10, 2, 128, 32, BF16, "int8", {"mean": True}),
    ([1], [40000], 8, 8, 64, 1024, BF16, "16bit", {}),
    ([1, 1], [20000, 3], 3, 1, 128, 64, F16, "int8", {}),
    ([70], [0], 4, 2, 64, 16, F16, "16bit", {}),
    ([200, 17], [333, 64], 8, 2, 128, 16, BF16, "16bit", {"layout": "NHD"}),
    ([200, 17], [333, 64], 8, 2, 128, 64, F16, "int8", {}),
    ([129, 1, 64, 0, 300], [0, 900, 65, 7, 1], 12, 4, 64, 32, BF16, "int8", {"mean": True}),
    ([257], [511], 6, 2, 128, 128, F16, "16bit", {}),
    ([1030], [77], 2, 2, 64, 256, F16, "16bit", {}),
    ([300, 40], [20, 3000], 7, 1, 128, 16, BF16, "16bit", {}),
    ([130], [130], 128, 1, 64, 16, F16, "16bit", {}),
    ([40], [200], 160, 1, 64, 16, BF16, "int8", {}),
    ([3, 2], [1000, 64], 20, 2, 128, 16, F16, "int8", {}),
    ([4, 1], [63, 700], 8, 1, 64, 64, BF16, "int8", {"layout": "NHD", "mean": True}),
    ([9], [2000], 24, 8, 128, 1024, F16, "16bit", {}),
    ([50], [3000], 200, 1, 128, 32, F16, "16bit", {}),
    # single tokens beside chunks: two kernels, each on its sequences
    ([1] * 19 + [200], [(i * 377) % 900 for i in range(20)], 8, 2, 128, 16, BF16, "16bit", {}),
    ([2, 1, 0, 1, 90, 1, 5, 4] + [1] * 10, [30, 0, 4, 700, 64, 63, 12, 1000] + [9] * 10, 8, 2, 64, 32, F16, "16bit", {}),
    ([1, 300, 2, 1, 1, 8, 0] + [1] * 30, [100, 0, 65, 3000, 1, 20, 3] + [77] * 30, 12, 2, 128, 64, BF16, "int8", {"mean": True}),
    ([1, 1, 40, 1, 1] + [1] * 20, [10, 20, 200, 640, 0] + [130] * 20, 20, 1, 64, 16, F16, "int8", {}),
]
MASKS = [dict(), dict(window=1), dict(window=50, sinks=4), dict(window=200, sinks=70), dict(window=64), dict(causal=False)]


def check(c, got, sm_scale=None, **mask):
    want, bound = attend(c, sm_scale=sm_scale, **mask)
    n = sum(c["new"])
    err = (got[:n].double() - want[:n]).abs()
    assert bool(got[:n].isfinite().all())
    worst = (err - bound[:n]).max().item() if n else 0
    print(f"max err {err.max().item():.2e}, {(err / bound[:n].clamp(min=1e-30)).max().item():.2f} of its bound")
    assert worst <= 0
    return want


@pytest.mark.parametrize("mask", MASKS, ids=str)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c)[:60])
def test_attention(case, mask):
    new, past, hq, hkv, dim, page, dtype, storage, opt = case
    c = make_case(DEV, new=new, past=past, hq=hq, hkv=hkv, dim=dim, page=page, dtype=dtype, storage=storage, seed=7, **opt)
    o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=c["max_new"], **mask)
    assert tb.device_status(DEV) == 0
    assert o.shape == c["q"].shape and o.dtype == dtype
    check(c, o, **mask)


def test_without_prefix_sums_every_sequence_has_one_token():
    c = make_case(DEV, new=[1] * 5, past=[3, 0, 70, 200, 64], hq=8, hkv=2, dim=128, page=16, dtype=BF16, seed=1)
    cache = cache_of(c)
    a = tb.run_paged_attn(c["q"], cache, c["table"], c["lens"], c["cu"], max_seqlen_q=1)
    b = tb.run_paged_attn(c["q"], cache, c["table"], c["lens"])
    assert torch.equal(a, b)
    check(c, a)


def test_a_query_that_sees_nothing_gives_zero():
    """More new tokens than the sequence holds: those before position 0 see no key; an empty sequence sees none."""
    c = make_case(DEV, new=[5, 3], past=[0, 20], hq=4, hkv=2, dim=64, page=16, dtype=F16, seed=2)
    lens = torch.tensor([2, 0], dtype=torch.int32, device=DEV)
    o = torch.full_like(c["q"], 9)
    tb.run_paged_attn(c["q"], cache_of(c), c["table"], lens, c["cu"], max_seqlen_q=5, out=o)
    assert bool((o[:3] == 0).all()) and bool((o[5:] == 0).all())
    small = dict(c, new=[2, 0], lens_host=[2, 0], lens=lens, q=c["q"][3:5], total=2)
    check(small, o[3:5])


@pytest.mark.parametrize("max_new", [1, 90])
def test_strided_queries_and_outputs_and_rows_behind_the_last_sequence(max_new):
    new = [1, 1, 1] if max_new == 1 else [90, 1, 30]
    c = make_case(DEV, new=new, past=[100, 30, 0], hq=6, hkv=2, dim=64, page=16, dtype=F16, seed=3, spare_rows=4)
    wide = torch.full((c["total"], 20, 64), 3.0, dtype=F16, device=DEV)
    q = wide[:, 2:8]
    q.copy_(c["q"])
    out = torch.full((6, c["total"], 64), 9.0, dtype=F16, device=DEV).transpose(0, 1)  # heads outside, tokens inside
    o = tb.run_paged_attn(q, cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=max_new, out=out, sm_scale=0.3)
    assert o is out
    check(c, o, sm_scale=0.3)
    assert bool((out[sum(new):] == 9).all())
    tb.run_paged_attn(q, cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=max_new, out=q, sm_scale=0.3)  # in place
    n = sum(new)
    assert torch.equal(q[:n], o[:n])


@pytest.mark.parametrize("n,hq", [(1, 2), (3, 16), (2, 8)])
@pytest.mark.parametrize("storage", ["16bit", "int8"])
def test_many_sequences(n, hq, storage):
    """More sequences than threads of a block, and more blocks of query rows than the schedule keeps at hand."""
    B = 2100
    c = make_case(DEV, new=[1 + i % n for i in range(B)], past=[i * 7 % 40 for i in range(B)], hq=hq, hkv=2, dim=64, page=16,
                  dtype=F16, storage=storage, seed=14)
    o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=n)
    check(c, o)
    # a larger bound on the new tokens, and so another kernel, changes roundings only
    o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"])
    check(c, o)


@pytest.mark.parametrize("n", [4, 100])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_hidden_keys_and_values_weigh_nothing(n, dtype):
    """The last token's key and value are the largest of the type: tokens before it do not notice."""
    c = make_case(DEV, new=[n], past=[150], hq=4, hkv=2, dim=128, page=16, dtype=dtype, seed=15)
    big = torch.finfo(dtype).max
    last = 150 + n - 1
    pg, row = int(c["table"][0, last // 16]), last % 16
    c["v"][pg, :, row] = big
    c["k"][pg, :, row] = torch.where(torch.rand(2, 128, device=DEV) < 0.5, -big, big).to(dtype)
    o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=n)
    want, bound = attend(c)
    assert bool(((o[:n - 1].double() - want[:n - 1]).abs() <= bound[:n - 1]).all())


@pytest.mark.parametrize("n", [1, 5, 100])
def test_unused_scales_may_hold_anything(n):
    for fill in (1e30, float("inf"), -5.0, 0.0):
        c = make_case(DEV, new=[n, n], past=[70, 5], hq=4, hkv=2, dim=64, page=32, dtype=F16, storage="int8", seed=16)
        for x in ("k_scale", "v_scale"):
            c["kw"][x].nan_to_num_(nan=fill)
        for mask in (dict(), dict(window=20, sinks=2)):
            o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=n, **mask)
            check(c, o, **mask)


def test_values_of_very_different_sizes_in_an_int8_cache():
    """The unit of the weights follows the largest scale seen; what came before it is rescaled."""
    for n in (1, 100):
        c = make_case(DEV, new=[n], past=[900], hq=4, hkv=2, dim=128, page=16, dtype=BF16, storage="int8", seed=17)
        s = c["kw"]["v_scale"]
        for j in range(0, 900 + n, 16):
            s[c["table"][0, j // 16].long()] *= 2.0 ** (j / 40 - 10)
        o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=n)
        check(c, o)


def test_a_slice_of_a_wider_page_table():
    c = make_case(DEV, new=[1, 40, 3], past=[100, 30, 0], hq=4, hkv=2, dim=64, page=16, dtype=F16, seed=18)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    w = c["table"].shape[1]
    wide[:, 7:7 + w] = c["table"]
    a, b = (tb.run_paged_attn(c["q"], cache_of(c), t, c["lens"], c["cu"], max_seqlen_q=40) for t in (c["table"], wide[:, 7:7 + w]))
    assert torch.equal(a, b)
    check(c, a)


def test_refusals_of_the_python_layer():
    c = make_case(DEV, new=[1, 2], past=[3, 0], hq=4, hkv=2, dim=64, page=16, dtype=F16, seed=19)
    cache = cache_of(c)
    q, table, lens, cu = c["q"], c["table"], c["lens"], c["cu"]
    kv = torch.zeros(3, 2, 64, dtype=F16, device=DEV)

    def attn(q=q, table=table, lens=lens, cu=cu, **kw):
        return tb.run_paged_attn(q, cache, table, lens, cu, **kw)

    for err, text, call in (
            (TypeError, "int32", lambda: attn(lens=lens.long())), (ValueError, "CUDA", lambda: attn(table=table.cpu())),
            (ValueError, "dimension", lambda: attn(table=table[0])), (ValueError, "batch", lambda: attn(lens=lens[:1])),
            (ValueError, "batch", lambda: attn(cu=cu[:2])), (ValueError, "columns", lambda: attn(table=table[:, :0])),
            (ValueError, "stride 1", lambda: attn(table=table.t().contiguous().t())),
            (TypeError, "dtype", lambda: attn(q=q.bfloat16())), (ValueError, "packed", lambda: attn(q=q[0])),
            (ValueError, "differs", lambda: attn(out=torch.zeros(5, 4, 64, dtype=F16, device=DEV))),
            (ValueError, "stride 1", lambda: attn(q=q.transpose(1, 2).contiguous().transpose(1, 2))),
            (ValueError, "window", lambda: attn(window=0)), (tb._native.SageError, "causal", lambda: attn(window=4, causal=False)),
            (tb._native.SageError, "window", lambda: attn(sinks=4)), (tb._native.SageError, "multiple", lambda: attn(q=q[:, :3])),
            (tb._native.SageError, "one token", lambda: attn(cu=None)), (tb._native.SageError, "overlaps k", lambda: attn(out=c["k"][:3, 0, :4])),
            (ValueError, "total", lambda: cache.gather(table, lens, cu)), (ValueError, "tokens", lambda: cache.append(kv, kv[:2], table, lens, cu)),
            (TypeError, "dtype", lambda: cache.append(kv.float(), kv, table, lens, cu)),
            (tb._native.SageError, "overlap", lambda: cache.gather(table, lens, cu, out=(kv, kv))),
            (ValueError, "one shape", lambda: tb.PagedKVCache(c["k"], c["v"][:1])),
            (TypeError, "int8", lambda: tb.PagedKVCache(c["k"].to(torch.int8), c["v"].to(torch.int8))),
            (ValueError, "belong", lambda: tb.PagedKVCache(c["k"], c["v"], k_mean=kv[0].float())),
            (tb._native.SageError, "page_size", lambda: tb.PagedKVCache.empty(4, 24, 2, 64, F16, DEV).append(kv, kv, table, lens, cu)),
            (tb._native.SageError, "head_dim", lambda: tb.PagedKVCache.empty(4, 16, 2, 32, F16, DEV).append(kv[..., :32], kv[..., :32], table, lens, cu)),
    ):
        with pytest.raises(err, match=text):
            call()
    assert tb.device_status(DEV) == 0


@pytest.mark.parametrize("storage", ["16bit", "int8"])
@pytest.mark.parametrize("n", [1, 100])
def test_extreme_values(storage, n):
    """Large scores (one key takes all the weight), values of very different sizes, and values near the type's largest."""
    for dtype, top in ((F16, 60000.0), (BF16, 2.0 ** 100)):
        c = make_case(DEV, new=[n], past=[300], hq=4, hkv=2, dim=128, page=16, dtype=dtype, storage=storage, seed=4)
        c["q"] *= 20
        if storage == "16bit":
            c["v"][::2] *= top / 8
            c["v"][1::2] *= 1e-3
        else:
            c["kw"]["v_scale"][::2] *= top / 8
            c["kw"]["v_scale"][1::2] *= 1e-5
        o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=n)
        check(c, o)


def test_same_inputs_give_the_same_bits():
    for n, storage in ((1, "16bit"), (1, "int8"), (120, "16bit"), (120, "int8")):
        c = make_case(DEV, new=[n, n], past=[5000, 33], hq=8, hkv=2, dim=128, page=16, dtype=BF16, storage=storage, seed=5)
        cache = cache_of(c)
        a, b = (tb.run_paged_attn(c["q"], cache, c["table"], c["lens"], c["cu"], max_seqlen_q=n) for _ in range(2))
        assert torch.equal(a, b)


def test_shared_pages():
    """Two sequences on the same pages (a shared prefix) and one page named twice."""
    c = make_case(DEV, new=[1, 1], past=[95, 95], hq=4, hkv=2, dim=64, page=16, dtype=F16, seed=6)
    c["table"][1] = c["table"][0]
    c["table"][1, 3] = c["table"][0, 2]
    o = tb.run_paged_attn(c["q"], cache_of(c), c["table"], c["lens"], c["cu"], max_seqlen_q=1)
    check(c, o)


@pytest.mark.parametrize("storage", ["16bit", "int8"])
def test_cache_past_32_bit_offsets(storage):
    """A cache of more than 2^31 elements (and bytes): the pages in use lie at its far end."""
    hkv, page, dim = 8, 64, 128
    pages = (1 << 31) // (hkv * page * dim) + 200
    cache = tb.PagedKVCache.empty(pages, page, hkv, dim, F16, DEV, storage=storage)
    new, past = [40, 1], [100, 300]
    c = make_case(DEV, new=new, past=past, hq=16, hkv=hkv, dim=dim, page=page, dtype=F16, storage=storage, seed=8)
    used = c["k"].shape[0]
    cache.k[-used:], cache.v[-used:] = c["k"], c["v"]
    if storage == "int8":
        cache.k_scale[-used:], cache.v_scale[-used:] = c["kw"]["k_scale"], c["kw"]["v_scale"]
    table = c["table"] + torch.where(c["table"] >= 0, pages - used, 0).to(torch.int32)
    o = tb.run_paged_attn(c["q"], cache, table, c["lens"], c["cu"], max_seqlen_q=40)
    check(c, o)
    a = tb.run_paged_attn(c["q"][:2], cache, table, c["lens"])
    check(dict(c, new=[1, 1], q=c["q"][:2], total=2), a)
    x = torch.randn(41, hkv, dim, device=DEV).half()
    cache.append(x, x, table, c["lens"], c["cu"])
    k, v = cache.gather(table, c["lens"], c["cu"], total=41)
    step = 0 if storage == "16bit" else x.float().abs().amax(-1, keepdim=True) / 254
    for t in (k, v):  # half a step of the code, and one rounding to 16 bits
        assert bool(((t.float() - x.float()).abs() <= (step + x.float().abs() * 2.0 ** -10) * (storage != "16bit")).all())


# ------------------------------------------------------------------ together, as a server uses them
@pytest.mark.parametrize("storage,mean", [("16bit", False), ("int8", True)])
def test_prompt_then_tokens(storage, mean):
    """A prompt arrives in two chunks, then single tokens: each step's output is attention over what was written."""
    hq, hkv, dim, page, dtype = 8, 2, 128, 16, BF16
    steps = [[40, 130], [25, 1], [1, 1], [1, 1], [3, 2]]
    total = [sum(s[b] for s in steps) for b in range(2)]
    km = torch.randn(hkv, dim, device=DEV) * 2 if mean else None
    cache = tb.PagedKVCache.empty(40, page, hkv, dim, dtype, DEV, storage=storage, k_mean=km)
    table = torch.randperm(40, device=DEV)[:24].to(torch.int32).view(2, 12)
    have = [0, 0]
    g = torch.Generator(device=DEV).manual_seed(9)
    assert max(total) <= 12 * page
    for s in steps:
        have = [a + b for a, b in zip(have, s)]
        n = sum(s)
        q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV) for h in (hq, hkv, hkv))
        if mean:
            k = k + km
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        lens = torch.tensor(have, dtype=torch.int32, device=DEV)
        cu = torch.tensor([0, s[0], n], dtype=torch.int32, device=DEV)
        cache.append(k, v, table, lens, cu)
        o = tb.run_paged_attn(q, cache, table, lens, cu, max_seqlen_q=max(s), window=60, sinks=2)
        kw = dict(tensor_layout="HND")
        if storage == "int8":
            kw.update(k_scale=cache.k_scale, v_scale=cache.v_scale, k_mean=km)
        c = dict(k=cache.k, v=cache.v, kw=kw, table=table, new=s, lens_host=have, q=q, total=n, dtype=dtype,
                 heads=(hq, hkv, dim), page=page)
        check(c, o, window=60, sinks=2)
        # the cache holds what was written: half a code step plus roundings of the sums and of the result
        row = 0
        for b, m in enumerate(s):
            kk, vv = held(c, b, have[b] - m, have[b])
            for got, x, off in ((kk, k, km), (vv, v, None)):
                x = x[row:row + m].double().transpose(0, 1)
                y = x if off is None else x - off.double()[:, None]
                tol = 0 if storage == "16bit" else y.abs().amax(-1, keepdim=True) / 127 * (0.5 + 127 * 2.0 ** -22) + 1e-6
                assert bool(((got - x).abs() <= tol).all())
            row += m


def test_matches_packed_flash_attention_on_a_whole_prompt():
    """A prompt with nothing before it is run_flash_attn_varlen's causal case."""
    new = [300, 65, 1]
    c = make_case(DEV, new=new, past=[0, 0, 0], hq=8, hkv=2, dim=128, page=32, dtype=F16, seed=11)
    cache = cache_of(c)
    k, v = (torch.randn(sum(new), 2, 128, device=DEV).half() for _ in range(2))
    cache.append(k, v, c["table"], c["lens"], c["cu"])
    a = tb.run_paged_attn(c["q"], cache, c["table"], c["lens"], c["cu"], max_seqlen_q=300)
    b = tb.run_flash_attn_varlen(c["q"], k, v, c["cu"], c["cu"], causal=True)
    want, bound = attend(c)
    assert bool(((a.double() - want).abs() <= bound).all())
    # both are within the bound of the same value, the packed kernel with its own exponential (2^-13 relative)
    assert bool(((a.double() - b.double()).abs() <= 2 * bound + 2.0 ** -12 * bound.amax() / 2.0 ** -11).all())


@pytest.mark.parametrize("n", [1, 64])
def test_captured_and_replayed_after_changes_in_place(n):
    """Two graphs (append + attention) over one cache, replayed in turn after lengths and tokens changed in place."""
    hq, hkv, dim, page = 8, 2, 64, 16
    cache = tb.PagedKVCache.empty(64, page, hkv, dim, F16, DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    sides = []
    for side in range(2):
        c = make_case(DEV, new=[n, n], past=[0, 0], hq=hq, hkv=hkv, dim=dim, page=page, dtype=F16, seed=side)
        st = dict(q=c["q"].clone(), k=torch.randn(2 * n, hkv, dim, device=DEV).half(), cu=c["cu"],
                  table=(torch.arange(32, **i32) + 32 * side).view(2, 16), lens=torch.tensor([n, n], **i32))
        st["v"] = torch.randn_like(st["k"])
        sides.append(st)

    def step(st):
        cache.append(st["k"], st["v"], st["table"], st["lens"], st["cu"])
        return tb.run_paged_attn(st["q"], cache, st["table"], st["lens"], st["cu"], max_seqlen_q=n)

    for st in sides:
        step(st)
    torch.cuda.synchronize(DEV)
    for st in sides:
        st["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(st["graph"]):
            st["o"] = step(st)
    for i in range(3):
        for st in sides:
            st["lens"].copy_(torch.tensor([n * (i + 1), n * (i + 1) + 7 * i], **i32))
            for x in ("q", "k", "v"):
                st[x].copy_(torch.randn_like(st[x]))
        for st in sides:
            st["graph"].replay()
        torch.cuda.synchronize(DEV)
        for st in sides:
            c = dict(k=cache.k.nan_to_num(0), v=cache.v.nan_to_num(0), kw=dict(tensor_layout="HND"), table=st["table"], new=[n, n],
                     lens_host=st["lens"].tolist(), q=st["q"], total=2 * n, dtype=F16, heads=(hq, hkv, dim), page=page)
            if i == 0:  # later steps leave positions unwritten that nothing filled
                check(c, st["o"])
            again = tb.run_paged_attn(st["q"], cache, st["table"], st["lens"], st["cu"], max_seqlen_q=n)
            assert torch.equal(again.nan_to_num(7), st["o"].nan_to_num(7))


def test_two_streams_at_once():
    c = make_case(DEV, new=[1] * 8, past=[900] * 8, hq=8, hkv=8, dim=128, page=16, dtype=BF16, seed=12)
    d = make_case(DEV, new=[64, 64], past=[700, 100], hq=8, hkv=8, dim=128, page=16, dtype=BF16, seed=13)
    caches = [cache_of(c), cache_of(d)]
    want = [tb.run_paged_attn(x["q"], y, x["table"], x["lens"], x["cu"], max_seqlen_q=x["max_new"])
            for x, y in zip((c, d), caches)]
    torch.cuda.synchronize(DEV)
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, (x, y) in enumerate(zip((c, d), caches)):
            with torch.cuda.stream(streams[i]):
                got[i].append(tb.run_paged_attn(x["q"], y, x["table"], x["lens"], x["cu"], max_seqlen_q=x["max_new"]))
    torch.cuda.synchronize(DEV)
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_empty_calls():
    cache = tb.PagedKVCache.empty(2, 16, 1, 64, F16, DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    none = torch.empty(0, 1, 64, dtype=F16, device=DEV)
    for batch in (0, 2):
        table, lens, cu = torch.zeros(batch, 1, **i32), torch.zeros(batch, **i32), torch.zeros(batch + 1, **i32)
        cache.append(none, none, table, lens, cu)
        assert cache.gather(table, lens, cu, total=0)[0].shape == (0, 1, 64)
        assert tb.run_paged_attn(none, cache, table, lens, cu).shape == (0, 1, 64)
