"""Plain 64-bit implementation of the paged cache operators, sequence by sequence, and random cases for them."""
import random

import torch


def make_case(device, *, new, past, hq=4, hkv=2, dim=64, page=16, dtype=torch.float16, storage="16bit", layout="HND",
              mean=False, seed=0, spare_rows=0, extra_cols=1):
    """Random cache contents, page table and queries. ``new`` / ``past``: tokens per sequence."""
    g = torch.Generator(device=device).manual_seed(seed)
    lens = [a + b for a, b in zip(new, past)]
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 3, max(need + [0]) + extra_cols
    order = torch.randperm(pages, generator=g, device=device)[:sum(need)].to(torch.int32).cpu()
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=device)

    full = (pages, hkv, page, dim)
    kw = {}
    if storage == "int8":
        k, v = (torch.randint(-127, 128, full, generator=g, device=device, dtype=torch.int8) for _ in range(2))
        kw = {x: (0.5 + torch.rand(full[:3], generator=g, device=device)) / 100 for x in ("k_scale", "v_scale")}
        kw["dtype"] = dtype
        if mean:
            kw["k_mean"] = randn(hkv, dim) * 2
    else:
        k, v = randn(*full).to(dtype), randn(*full).to(dtype)
    # what no position of a sequence reaches holds NaN
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(need[b]):
            used[table[b, j], :min(page, n - j * page)] = True
    free = ~used.to(device)[:, None, :].expand(pages, hkv, page)
    if storage == "int8":
        kw["k_scale"][free] = float("nan")
        kw["v_scale"][free] = float("nan")
    else:
        k[free] = float("nan")
        v[free] = float("nan")
    if layout == "NHD":
        k, v = (t.transpose(1, 2).contiguous() for t in (k, v))
    total = sum(new) + spare_rows
    cu = torch.tensor([0] + list(new)).cumsum(0).to(torch.int32)
    return dict(k=k, v=v, kw=dict(kw, tensor_layout=layout), table=table.to(device), lens=torch.tensor(lens, dtype=torch.int32, device=device),
                cu=cu.to(device), new=list(new), lens_host=lens, q=randn(total, hq, dim).to(dtype), total=total, dtype=dtype,
                heads=(hq, hkv, dim), page=page, max_new=max(list(new) + [1]))


def held(c, b, lo, hi, with_mean=True):
    """Keys and values of positions [lo, hi) of sequence b in 64 bits: [hkv, hi - lo, dim]."""
    pos = torch.arange(lo, hi, device=c["k"].device)
    pg, row = c["table"][b].long()[pos // c["page"]], pos % c["page"]
    k, v = c["k"], c["v"]
    if c["kw"]["tensor_layout"] == "NHD":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    k, v = k[pg, :, row].double(), v[pg, :, row].double()
    if "k_scale" in c["kw"]:
        k = k * c["kw"]["k_scale"][pg, :, row].double()[..., None]
        v = v * c["kw"]["v_scale"][pg, :, row].double()[..., None]
        if with_mean and c["kw"].get("k_mean") is not None:
            k = k + c["kw"]["k_mean"].double()
    return k.transpose(0, 1), v.transpose(0, 1)


def attend(c, *, causal=True, window=None, sinks=0, sm_scale=None):
    """(o, bound): the definition in 64 bits and how far a kernel may be from it, elementwise.

    bound: the kernel rounds each weight to 16 bits (relative u = eps / 2 of the type, or 2^-25 of the largest
    weight where fp16 turns subnormal; of the largest weight times v_scale and per code in an int8 cache), accumulates in fp32 and rounds the result once: with A = sum_j w_j |v_j|
    (w: the softmax), |err| <= u A + u |o| + 2^-25 sum_j |v_j| / (sum of weights, >= 1) + e A. e: relative error of
    a weight and of its sum beyond the rounding: twice the error of a score, which is (dim / 16 + 8) products'
    accumulation roundings of 2^-23 of sum |q k| (bf16 queries of an int8 cache: also 2^-24 of the largest
    |q| times sum |k|), plus 2^-20 for the exponential and scales, plus 2^-23 per accumulated group of 16 keys.
    """
    hq, hkv, dim = c["heads"]
    g = hq // hkv
    scale = dim ** -0.5 if sm_scale is None else sm_scale
    u = torch.finfo(c["dtype"]).eps / 2
    o = torch.zeros(c["total"], hq, dim, dtype=torch.float64, device=c["k"].device)
    bound = torch.zeros_like(o)
    row = 0
    for b, n in enumerate(c["new"]):
        L = c["lens_host"][b]
        if n and L:
            k, v = held(c, b, 0, L, with_mean=False)
            q = c["q"][row:row + n].double().view(n, hkv, g, dim).permute(1, 2, 0, 3).reshape(hkv, g * n, dim)
            pos = (torch.arange(n, device=k.device) + L - n).repeat(g)[:, None]
            key = torch.arange(L, device=k.device)[None]
            see = key <= pos if causal else (key >= 0).expand(g * n, L)
            if window:
                see = see & ((key > pos - window) | (key < sinks))
            s = (q @ k.transpose(1, 2)) * scale
            size = ((q.abs() @ k.abs().transpose(1, 2)) * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
            low = (q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None] * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
            s = s.masked_fill(~see, float("-inf"))
            top = s.amax(-1, keepdim=True)
            top = torch.where(top.isfinite(), top, torch.zeros_like(top))
            e = torch.exp(s - top)
            z = e.sum(-1, keepdim=True)
            w = torch.where(z > 0, e / z, torch.zeros_like(e))
            out, big = w @ v, w @ v.abs()
            tiny = see.double() @ v.abs() / z.clamp(min=1)
            if "v_scale" in c["kw"]:
                at = torch.arange(L, device=k.device)
                vs = c["kw"]["v_scale"][c["table"][b].long()[at // c["page"]], :, at % c["page"]].double().t()  # [hkv, L]
                code = v.abs() / vs[..., None].clamp(min=1e-300)
                tiny = torch.maximum(tiny, (w * vs[:, None]).amax(-1, keepdim=True) * (see.double() @ code))
            slack = 2 * ((dim / 16 + 8) * 2.0 ** -23 * size + 2.0 ** -24 * low) + 2.0 ** -20 + 2.0 ** -23 * (L / 16 + 16)
            bd = (u + slack) * big + u * out.abs() + 2.0 ** -25 * tiny

            def rows(x):
                return x.view(hkv, g, n, dim).permute(2, 0, 1, 3).reshape(n, hq, dim)

            o[row:row + n], bound[row:row + n] = rows(out), rows(bd)
        row += n
    return o, bound


def log_lengths(rng: random.Random, lo, hi, n):
    return [int(round(lo * (hi / lo) ** rng.random())) for _ in range(n)]
