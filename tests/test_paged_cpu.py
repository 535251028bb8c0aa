"""CPU: argument checks of the paged cache's C entry points (no GPU call is made) and of its Python layer, and the plain
implementation that the GPU tests compare with, against an elementary one."""
import ctypes

import pytest
import torch

import tribench_b200 as tb
from paged_ref import attend, make_case
from tribench_b200 import _native as N

KEEP = []


def buf(n=1 << 16):
    b = (ctypes.c_uint8 * (n + 256))()
    KEEP.append(b)
    return (ctypes.addressof(b) + 255) & ~255


@pytest.fixture(scope="module")
def ptr():
    return {n: buf() for n in ("k", "v", "ks", "vs", "km", "q", "o", "nk", "nv", "table", "lens", "cu", "ws")}


def cache(ptr, **kw):
    storage = kw.pop("storage", N.SAGE_CACHE_16BIT)
    i8 = storage == N.SAGE_CACHE_INT8
    f = dict(k=ptr["k"], v=ptr["v"], k_scale=ptr["ks"] if i8 else None, v_scale=ptr["vs"] if i8 else None, k_mean=None, num_pages=4,
             page_size=16, heads_kv=2, head_dim=64, k_strides=(2048, 1024, 64), v_strides=(2048, 1024, 64),
             dtype=N.SAGE_DTYPE_F16, storage=storage)
    f.update(kw)
    for x in ("k_strides", "v_strides"):
        f[x] = (ctypes.c_int64 * 3)(*f[x])
    return N.PagedCacheStruct(**f)


S2 = (64, 128)


def attn(ptr, c=None, lib=None, **kw):
    a = dict(q=ptr["q"], qs=(64, 256), o=ptr["o"], os=(64, 256), hq=4, table=ptr["table"], stride=4, width=4, lens=ptr["lens"],
             cu=ptr["cu"], batch=2, total=6, max_q=3, causal=1, window=0, sinks=0, ws=ptr["ws"], wsn=1 << 40)
    a.update(kw)
    c = c or cache(ptr)
    return N.load().sage_paged_attn_fwd(ctypes.byref(c), a["q"], N.strides2(*a["qs"]), a["o"], N.strides2(*a["os"]), a["hq"],
                                        a["table"], a["stride"], a["width"], a["lens"], a["cu"], a["batch"], a["total"], a["max_q"],
                                        a["causal"], a["window"], a["sinks"], 0.0, a["ws"], a["wsn"], None)


def move(ptr, fn="sage_paged_append", c=None, **kw):
    a = dict(k=ptr["nk"], v=ptr["nv"], ks=S2, vs=S2, table=ptr["table"], stride=4, width=4, lens=ptr["lens"], cu=ptr["cu"], batch=2,
             tokens=6)
    a.update(kw)
    c = c or cache(ptr)
    return getattr(N.load(), fn)(ctypes.byref(c), a["k"], a["v"], N.strides2(*a["ks"]), N.strides2(*a["vs"]), a["table"], a["stride"],
                                 a["width"], a["lens"], a["cu"], a["batch"], a["tokens"], None)


def refused(rc, text, code=N.SAGE_ERR_INVALID_ARG):
    msg = N.load().sage_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def test_the_struct_is_the_headers():
    # 5 pointers, 4 sizes, 2 x 3 strides, 2 ints
    assert ctypes.sizeof(N.PagedCacheStruct) == 5 * 8 + 4 * 8 + 6 * 8 + 2 * 4


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=7), "dtype"), (dict(storage=5), "storage"), (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"), (dict(num_pages=0), "num_pages"),
    (dict(heads_kv=0), "heads_kv"), (dict(k_strides=(2048, 1024, 60)), "stride"), (dict(v_strides=(2048, -8, 64)), "stride"),
    (dict(k=None), "NULL"), (dict(k_mean=1 << 20), "INT8"), (dict(k_scale=1 << 20), "INT8"),
    (dict(storage=N.SAGE_CACHE_INT8, k_scale=None), "NULL"), (dict(storage=N.SAGE_CACHE_INT8, k_strides=(2048, 1024, 72)), "stride"),
    (dict(k=8 + (1 << 20)), "aligned"),
])
def test_bad_caches_are_refused(ptr, kw, text):
    c = cache(ptr, **kw)
    refused(attn(ptr, c), text)
    refused(move(ptr, c=c), text)
    refused(move(ptr, "sage_paged_gather", c=c), text)


@pytest.mark.parametrize("kw,text", [
    (dict(table=None), "NULL"), (dict(lens=None), "NULL"), (dict(batch=-1), "batch"), (dict(width=0), "pages_per_seq"),
    (dict(stride=3), "table_stride"), (dict(cu=None), "one token"), (dict(cu=(1 << 20) + 2), "aligned"),
])
def test_bad_sequence_arrays_are_refused(ptr, kw, text):
    refused(attn(ptr, **kw), text)
    refused(move(ptr, **kw), text)
    refused(move(ptr, "sage_paged_gather", **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(hq=5), "multiple"), (dict(hq=0), "multiple"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
    (dict(window=4, causal=0), "causal"), (dict(sinks=4), "window"), (dict(max_q=0), "max_seqlen_q"), (dict(qs=(60, 256)), "stride"),
    (dict(os=(64, 0)), "stride"), (dict(q=None), "NULL"), (dict(o=8 + (1 << 20)), "aligned"), (dict(total=(1 << 30) + 1), "tokens"),
])
def test_bad_attention_arguments_are_refused(ptr, kw, text):
    refused(attn(ptr, **kw), text)


def test_workspace_and_overlaps_are_checked(ptr):
    refused(attn(ptr, wsn=16), "workspace", N.SAGE_ERR_WORKSPACE)
    refused(attn(ptr, ws=None), "workspace", N.SAGE_ERR_WORKSPACE)
    refused(attn(ptr, ws=ptr["ws"] + 4), "aligned")
    refused(attn(ptr, o=ptr["k"] + 64, wsn=1 << 15 << 20), "overlaps k")
    refused(attn(ptr, o=ptr["q"] + 16), "overlaps q")
    refused(move(ptr, k=ptr["v"] + 32), "overlaps the cache")
    refused(move(ptr, "sage_paged_gather", v=ptr["nk"] + 64), "overlap each other")
    i8 = cache(ptr, storage=N.SAGE_CACHE_INT8)
    refused(move(ptr, "sage_paged_gather", c=i8, k=ptr["ks"]), "overlaps the cache")
    # a valid call passes every check and stops at the missing device
    if not torch.cuda.is_available():
        n = N.load().sage_paged_workspace_bytes(ctypes.byref(cache(ptr)), 4, 2, 6, 3, 4)
        for rc in (attn(ptr, ws=buf(n), wsn=n), attn(ptr, ws=buf(n), wsn=n, o=ptr["q"]), move(ptr), move(ptr, "sage_paged_gather")):
            assert rc not in (N.SAGE_OK, N.SAGE_ERR_INVALID_ARG, N.SAGE_ERR_WORKSPACE)


def test_workspace_covers_every_kernel_of_a_call(ptr):
    """Few rows: a size of its own; many: one that grows with the blocks of rows; a mixed batch: the larger of the two."""
    c = cache(ptr, head_dim=128, k_strides=(4096, 2048, 128), v_strides=(4096, 2048, 128))

    def size(hq, batch, total, max_q):
        return N.load().sage_paged_workspace_bytes(ctypes.byref(c), hq, batch, total, max_q, 64)

    few = size(8, 32, 32, 1)
    assert few > 0 and few == size(8, 1000, 2000, 2) == size(16, 1, 2, 2)
    many = size(8, 2, 1000, 600)
    assert size(8, 2, 100000, 60000) > many
    mixed = size(8, 64, 63 + 512, 512)
    assert mixed >= few and mixed >= size(8, 2, 63 + 512, 512)
    for bad in ((0, 1, 1, 1), (8, 0, 1, 1), (8, 1, 0, 1), (8, 1, 1, 0), (3, 1, 1, 1)):
        assert size(*bad) == 0


def test_empty_calls_do_nothing(ptr):
    assert attn(ptr, total=0) == N.SAGE_OK and attn(ptr, batch=0, total=0, cu=None, table=None, lens=None) == N.SAGE_OK
    assert move(ptr, tokens=0) == N.SAGE_OK and move(ptr, "sage_paged_gather", tokens=0) == N.SAGE_OK


def test_python_layer_refuses_host_tensors_and_wrong_types():
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        tb.PagedKVCache(k, k)
    with pytest.raises(TypeError, match="torch.Tensor"):
        tb.PagedKVCache([1], k)
    with pytest.raises(ValueError, match="storage"):
        tb.PagedKVCache.empty(2, 16, 1, 64, torch.float16, "cpu", storage="int4")
    with pytest.raises(TypeError, match="dtype"):
        tb.PagedKVCache.empty(2, 16, 1, 64, torch.float32, "cpu")
    with pytest.raises(TypeError, match="PagedKVCache"):
        tb.run_paged_attn(k, None, None, None)


@pytest.mark.parametrize("storage", ["16bit", "int8"])
@pytest.mark.parametrize("mask", [dict(), dict(window=5, sinks=2), dict(causal=False)], ids=str)
def test_plain_implementation(storage, mask):
    """paged_ref.attend, row by row and key by key."""
    c = make_case("cpu", new=[3, 0, 1, 4], past=[20, 5, 0, 13], hq=4, hkv=2, dim=64, page=16, storage=storage, seed=1)
    got, bound = attend(c, **mask)
    row = 0
    for b, n in enumerate(c["new"]):
        L = c["lens_host"][b]
        for i in range(n):
            p = L - n + i
            keys = [j for j in range(L) if mask.get("causal") is False or (j <= p and (
                "window" not in mask or j > p - mask["window"] or j < mask["sinks"]))]
            for h in range(4):
                ks, vs = [], []
                for j in keys:
                    pg, r = int(c["table"][b, j // 16]), j % 16
                    k, v = c["k"][pg, h // 2, r].double(), c["v"][pg, h // 2, r].double()
                    if storage == "int8":
                        k, v = k * c["kw"]["k_scale"][pg, h // 2, r].double(), v * c["kw"]["v_scale"][pg, h // 2, r].double()
                    ks.append(k), vs.append(v)
                s = torch.stack(ks) @ c["q"][row + i, h].double() / 8
                w = torch.softmax(s, 0)
                assert (w @ torch.stack(vs) - got[row + i, h]).abs().max() < 1e-12
        row += n
    assert bool(got.isfinite().all()) and bool((bound[:row] >= 0).all())
