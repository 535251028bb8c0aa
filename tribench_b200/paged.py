"""Paged key/value cache and attention over it: the serving side of the attention operators.

The reference's packs attend over whole [B, H, S, D] tensors (kernels/flash_attn/triton_impl.py:110-128,
kernels/sage_attn/triton_impl.py:162-200) and hold no cache; these operators extend them to tokens that
arrive one by one or chunk by chunk.

A cache holds keys and values of many sequences in pages of ``page_size`` tokens. Which page holds what
is the caller's: ``page_table`` [batch, pages_per_seq] (int32) names the pages of each sequence in order,
and ``seq_lens`` [batch] (int32) says how many tokens each holds, the new ones of the call included.
New tokens are packed along one axis, [tokens, heads, head_dim], as in varlen.py; ``cu_seqlens`` (int32
prefix sums of their numbers, [batch + 1]) says whose they are, or None: one token per sequence. New
token i of the n of sequence b has position ``seq_lens[b] - n + i``.

    cache = PagedKVCache.empty(num_pages, 64, heads_kv, head_dim, torch.bfloat16, "cuda", storage="int8")
    cache.append(k, v, page_table, seq_lens, cu_seqlens)          # the new tokens' keys and values
    o = run_paged_attn(q, cache, page_table, seq_lens, cu_seqlens, max_seqlen_q=512)

All three arrays stay on the device: no call reads them on the host, waits, or depends on their values
in its launches, so calls can be captured into CUDA graphs and replayed after the arrays (and the
tokens) were changed in place. They are not validated on the host for the same reason; the kernels keep
every access inside the tensors whatever they hold (see the C header).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import torch

from . import _native as N
from .sage_attn import _DTYPES, _check_tensor


# A step of a small model makes hundreds of these calls, so what runs on the host per call is kept
# short: stride arrays and workspace sizes are looked up by value, the stream and the current device
# are asked for directly.
_strides2 = functools.lru_cache(maxsize=1024)(N.strides2)


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


_HERE = contextlib.nullcontext()


def _on(device):
    """Context with ``device`` current."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _packed2(name: str, t: torch.Tensor, heads: int, dim: int, dtype, device):
    """Checks a packed [tokens, heads, dim] tensor; (tokens, element strides {head, token})."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device:
        _check_tensor(name, t, dtype)
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{name} must be a packed [tokens, {heads}, {dim}] tensor, got shape {tuple(shape)}")
    st, sh, sd = t.stride()
    if sd != 1:
        raise ValueError(f"{name}: the head dimension must be contiguous (stride 1)")
    # the stride of an axis of one entry is never used: any valid one serves
    return shape[0], _strides2(sh if heads > 1 else dim, st if shape[0] > 1 else heads * dim)


def _seqs(page_table, seq_lens, cu_seqlens, device):
    """Checks the page table, lengths and prefix sums of a call; (table, its row stride, pages per sequence, lens, cu,
    batch) as the C entry points take them."""
    for name, t in (("page_table", page_table), ("seq_lens", seq_lens), ("cu_seqlens", cu_seqlens)):
        if t is None and name == "cu_seqlens":
            continue
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.device != device:
            _check_tensor(name, t, torch.int32)
            raise ValueError(f"{name} is on {t.device}, the cache on {device}")
        dims = 2 if name == "page_table" else 1
        if t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimension(s), got shape {tuple(t.shape)}")
    batch, width = page_table.shape
    if width == 0:
        raise ValueError("page_table has no columns")
    stride, inner = page_table.stride()
    if width > 1 and inner != 1:
        raise ValueError("page_table: the pages of a sequence must be contiguous (stride 1)")
    if seq_lens.shape[0] != batch or (batch > 1 and seq_lens.stride(0) != 1):
        raise ValueError(f"seq_lens must be a contiguous vector of batch = {batch} entries")
    if cu_seqlens is not None and (cu_seqlens.shape[0] != batch + 1 or cu_seqlens.stride(0) != 1):
        raise ValueError(f"cu_seqlens must be a contiguous vector of batch + 1 = {batch + 1} entries")
    return (page_table.data_ptr(), stride if batch > 1 else width, width, seq_lens.data_ptr(),
            None if cu_seqlens is None else cu_seqlens.data_ptr(), batch)


class PagedKVCache:
    """Keys and values in pages, over the caller's tensors.

    ``k``, ``v``: [num_pages, heads_kv, page_size, head_dim] (``tensor_layout="HND"``) or
    [num_pages, page_size, heads_kv, head_dim] ("NHD"), any strides that are multiples of 16 bytes with a
    contiguous head dimension; float16 / bfloat16 values, or int8 codes. page_size: a power of two from
    16 to 1024; head_dim 64 or 128.

    int8 codes need ``k_scale`` and ``v_scale`` ([num_pages, heads_kv, page_size] float32, contiguous,
    whatever the layout: one scale per token and head) and ``dtype``, the 16-bit type of new tokens, of
    tokens read back and of attention. Row x is held as scale = max|x| / 127 and codes
    rint(127 x / max|x|). ``k_mean`` ([heads_kv, head_dim] float32, optional) is subtracted from keys
    before they are quantised and added when they are read back, the cache's form of the smoothing of
    run_sage_attn: keys share large channel offsets that would use up the codes' range, and a constant
    offset of all keys does not change attention. It must stay the same for the cache's life.

    The tensors and sizes are fixed: the calls use the addresses of construction, so neither the
    attributes nor the tensors' storages can be exchanged (their contents can).
    """

    _FIXED = frozenset(("k", "v", "k_scale", "v_scale", "k_mean", "dtype", "device", "tensor_layout", "storage", "num_pages",
                        "heads_kv", "page_size", "head_dim"))

    def __setattr__(self, name, value):
        if name in self._FIXED and "_c" in self.__dict__:
            raise AttributeError(f"PagedKVCache.{name} is fixed: make another cache for other tensors")
        object.__setattr__(self, name, value)

    def __init__(self, k, v, *, k_scale=None, v_scale=None, k_mean=None, dtype=None, tensor_layout="HND"):
        _check_tensor("k", k)
        _check_tensor("v", v, k.dtype)
        if v.device != k.device:
            raise ValueError(f"v is on {v.device}, k on {k.device}")
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError(f"k and v must be 4-D tensors of one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("the head dimension must be contiguous (stride 1)")
        if tensor_layout == "HND":
            axes = (0, 1, 2)
        elif tensor_layout == "NHD":
            axes = (0, 2, 1)
        else:
            raise ValueError(f"tensor_layout must be 'HND' or 'NHD', got {tensor_layout!r}")
        pages, heads, page, dim = *(k.shape[a] for a in axes), k.shape[3]
        self.storage = "int8" if k.dtype == torch.int8 else "16bit"
        if self.storage == "int8":
            if dtype not in _DTYPES:
                raise TypeError(f"an int8 cache needs dtype float16 or bfloat16, got {dtype}")
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                _check_tensor(name, t, torch.float32)
                if tuple(t.shape) != (pages, heads, page) or not t.is_contiguous() or t.device != k.device:
                    raise ValueError(f"{name} must be a contiguous ({pages}, {heads}, {page}) tensor on {k.device}")
            if k_mean is not None:
                _check_tensor("k_mean", k_mean, torch.float32)
                if tuple(k_mean.shape) != (heads, dim) or not k_mean.is_contiguous() or k_mean.device != k.device:
                    raise ValueError(f"k_mean must be a contiguous ({heads}, {dim}) tensor on {k.device}")
        else:
            if k.dtype not in _DTYPES:
                raise TypeError(f"k/v must be float16, bfloat16 or int8, got {k.dtype}")
            if dtype not in (None, k.dtype):
                raise TypeError(f"dtype {dtype} differs from the cache's {k.dtype}")
            if k_scale is not None or v_scale is not None or k_mean is not None:
                raise ValueError("scales and k_mean belong to an int8 cache")
            dtype = k.dtype
        self.k, self.v, self.k_scale, self.v_scale, self.k_mean = k, v, k_scale, v_scale, k_mean
        self.dtype, self.device, self.tensor_layout = dtype, k.device, tensor_layout
        self.num_pages, self.heads_kv, self.page_size, self.head_dim = pages, heads, page, dim

        def strides(t):
            full = (heads * page * dim, page * dim, dim)  # for axes of one entry, whose stride is never used
            return (ctypes.c_int64 * 3)(*(t.stride(a) if t.shape[a] > 1 else f for a, f in zip(axes, full)))

        def ptr(t):
            return None if t is None else t.data_ptr()

        self._c = N.PagedCacheStruct(ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), ptr(k_mean), pages, page, heads, dim,
                                     strides(k), strides(v), _DTYPES[dtype],
                                     N.SAGE_CACHE_INT8 if self.storage == "int8" else N.SAGE_CACHE_16BIT)
        self._ref = ctypes.byref(self._c)
        self._lib = N.load()
        self._workspace = functools.lru_cache(maxsize=256)(functools.partial(self._lib.sage_paged_workspace_bytes, self._ref))

    @classmethod
    def empty(cls, num_pages, page_size, heads_kv, head_dim, dtype, device, *, storage="16bit", tensor_layout="HND",
              k_mean=None):
        """A cache with tensors of its own, their contents unset. ``storage``: "16bit" or "int8"."""
        if storage not in ("16bit", "int8"):
            raise ValueError(f"storage must be '16bit' or 'int8', got {storage!r}")
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be float16 or bfloat16, got {dtype}")
        shape = (num_pages, heads_kv, page_size, head_dim)
        if tensor_layout == "NHD":
            shape = (num_pages, page_size, heads_kv, head_dim)
        kind = torch.int8 if storage == "int8" else dtype
        k, v = (torch.empty(shape, dtype=kind, device=device) for _ in range(2))
        scales = {}
        if storage == "int8":
            scales = {x: torch.empty((num_pages, heads_kv, page_size), dtype=torch.float32, device=device)
                      for x in ("k_scale", "v_scale")}
        return cls(k, v, **scales, k_mean=k_mean, dtype=dtype, tensor_layout=tensor_layout)

    def append(self, k, v, page_table, seq_lens, cu_seqlens=None):
        """Write the new tokens' keys and values ([tokens, heads_kv, head_dim] in the cache's dtype).

        No two new tokens of a call may name the same place (two sequences that write into a shared page)."""
        tokens, ks = _packed2("k", k, self.heads_kv, self.head_dim, self.dtype, self.device)
        tv, vs = _packed2("v", v, self.heads_kv, self.head_dim, self.dtype, self.device)
        if tv != tokens:
            raise ValueError(f"k has {tokens} tokens, v {tv}")
        s = _seqs(page_table, seq_lens, cu_seqlens, self.device)
        with _on(self.device):
            rc = self._lib.sage_paged_append(self._ref, k.data_ptr(), v.data_ptr(), ks, vs, *s, tokens,
                                             _raw_stream(self.device.index))
        if rc:
            N.check("sage_paged_append", rc)

    def gather(self, page_table, seq_lens, cu_seqlens=None, *, total=None, out=None):
        """Read the newest tokens of each sequence back: (k, v), each [tokens, heads_kv, head_dim].

        ``cu_seqlens`` says how many of each (all of sequence b's: a difference of ``seq_lens[b]``);
        ``total`` is its last entry, which the host has to know to allocate the result (default without
        cu_seqlens: one per sequence). ``out``: a pair of tensors to write into instead. Rows behind the
        last sequence are left as they are."""
        s = _seqs(page_table, seq_lens, cu_seqlens, self.device)
        if out is None:
            if total is None:
                if cu_seqlens is not None:
                    raise ValueError("gather needs total (the number of tokens) or out")
                total = s[-1]
            shape = (int(total), self.heads_kv, self.head_dim)
            k = torch.empty(shape, dtype=self.dtype, device=self.device)
            v = torch.empty(shape, dtype=self.dtype, device=self.device)
        else:
            k, v = out
        tokens, ks = _packed2("out[0]", k, self.heads_kv, self.head_dim, self.dtype, self.device)
        tv, vs = _packed2("out[1]", v, self.heads_kv, self.head_dim, self.dtype, self.device)
        if tv != tokens or (total is not None and tokens != int(total)):
            raise ValueError(f"out holds {tokens} and {tv} tokens, expected {tokens if total is None else int(total)}")
        with _on(self.device):
            rc = self._lib.sage_paged_gather(self._ref, k.data_ptr(), v.data_ptr(), ks, vs, *s, tokens,
                                             _raw_stream(self.device.index))
        if rc:
            N.check("sage_paged_gather", rc)
        return k, v


def run_paged_attn(q, cache: PagedKVCache, page_table, seq_lens, cu_seqlens_q=None, max_seqlen_q=None, *, causal=True,
                   window=None, sinks=0, sm_scale=None, out=None):
    """Attention of new tokens over a cache that already holds their keys and values.

    q: [total_q, heads_q, head_dim] in the cache's dtype, heads_q a multiple of the cache's heads_kv.
    The query at position p of its sequence sees key j when j <= p (``causal``; else every key that the
    sequence holds) and, with ``window``, j > p - window or j < ``sinks``: the last ``window`` keys, its
    own among them, and the first ``sinks`` ones of the sequence. A query that sees nothing gets o = 0.
    ``max_seqlen_q``: the most new tokens of a sequence (default: total_q, or 1 without
    ``cu_seqlens_q``); it picks the kernels, so give it where it is known, and never less than it is (the
    rows of a sequence that has more are wrong). sm_scale defaults to head_dim ** -0.5. Returns o like q (written into ``out`` when given; ``out=q`` is allowed). The
    scratch of work split along the keys is allocated per call, so calls on several streams or in
    several graphs share nothing.
    """
    if not isinstance(cache, PagedKVCache):
        raise TypeError("cache must be a PagedKVCache")
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        _check_tensor("q", q, cache.dtype)
        raise ValueError(f"q must be a packed [tokens, heads, head_dim] tensor, got shape {tuple(q.shape)}")
    device, dim = cache.device, cache.head_dim
    heads = q.shape[1]
    total, qs = _packed2("q", q, heads, dim, cache.dtype, device)
    s = _seqs(page_table, seq_lens, cu_seqlens_q, device)
    if out is None:
        out = torch.empty((total, heads, dim), dtype=cache.dtype, device=device)
    to, os_ = _packed2("out", out, heads, dim, cache.dtype, device)
    if to != total:
        raise ValueError(f"out shape {tuple(out.shape)} differs from q {tuple(q.shape)}")
    if max_seqlen_q is None:
        max_seqlen_q = max(total, 1) if cu_seqlens_q is not None else 1
    if window is None:
        window = 0
    elif window <= 0:
        raise ValueError(f"window must be positive, got {window}")
    with _on(device):
        n = cache._workspace(heads, s[-1], total, max_seqlen_q, s[2])
        ws = torch.empty(n or 1, dtype=torch.uint8, device=device)
        rc = cache._lib.sage_paged_attn_fwd(cache._ref, q.data_ptr(), qs, out.data_ptr(), os_, heads, *s, total, max_seqlen_q,
                                            1 if causal else 0, window, sinks, 0.0 if sm_scale is None else sm_scale,
                                            ws.data_ptr(), n, _raw_stream(device.index))
    if rc:
        N.check("sage_paged_attn_fwd", rc)
    return out
