"""Work of the paged key/value cache operators: what a serving loop asks of them, and their plain form.

Three operators: writing new tokens into a paged cache (16 bit, or INT8 with one scale per token and
head), reading tokens back, and attention of new query tokens over the cache (single tokens, chunks,
whole prompts, mixed batches; causal, optionally with a sliding window and sinks).

Positions: sequence b holds lens[b] tokens after its n_b newest ones arrived; newest token i has
position lens[b] - n_b + i. Position p lives in page page_table[b, p // page], row p % page.
"""
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one generated token of each of 64 sequences is written: latency of a launch
        dict(name="write_tokens_bf16", op="write", batch=64, new_lo=1, new_hi=1, past_lo=100, past_hi=8000, hkv=8,
             dim=128, page=16, type="bf16", store="16bit", mean=False, mix=1),
        # prompts of very different lengths are quantised into the cache and read back
        dict(name="write_read_prompts_int8", op="write", batch=6, new_lo=37, new_hi=9001, past_lo=0, past_hi=0, hkv=8,
             dim=128, page=32, type="fp16", store="int8", mean=True, mix=2),
        # a long quantised cache is read back (prefix handed to another worker)
        dict(name="read_int8_bf16", op="read", batch=8, new_lo=501, new_hi=16384, past_lo=0, past_hi=0, hkv=8, dim=128,
             page=64, type="bf16", store="int8", mean=False, mix=3),
        # the newest tokens of every sequence in a 16-bit cache, small heads
        dict(name="read_tail_fp16_d64", op="read", batch=32, new_lo=1, new_hi=700, past_lo=0, past_hi=4096, hkv=4,
             dim=64, page=16, type="fp16", store="16bit", mean=False, mix=4),
        # a single conversation's next token, short context: latency
        dict(name="token_short_fp16", op="attend", batch=1, new_lo=1, new_hi=1, past_lo=700, past_hi=700, hq=32, hkv=8,
             dim=128, page=16, type="fp16", store="16bit", mean=False, window=0, sinks=0, mix=5),
        # the next token of a full batch, ragged contexts: cache bandwidth
        dict(name="token_batch_bf16", op="attend", batch=64, new_lo=1, new_hi=1, past_lo=200, past_hi=8191, hq=32, hkv=8,
             dim=128, page=16, type="bf16", store="16bit", mean=False, window=0, sinks=0, mix=6),
        # long contexts in a quantised cache, a wide head group
        dict(name="token_long_int8_bf16", op="attend", batch=16, new_lo=1, new_hi=1, past_lo=9000, past_hi=32767, hq=64,
             hkv=8, dim=128, page=64, type="bf16", store="int8", mean=True, window=0, sinks=0, mix=7),
        # streaming: a window and four sinks over long contexts, one draft of four tokens to verify
        dict(name="tokens_window_fp16_d64", op="attend", batch=32, new_lo=4, new_hi=4, past_lo=5000, past_hi=32000, hq=16,
             hkv=16, dim=64, page=32, type="fp16", store="16bit", mean=False, window=4096, sinks=4, mix=8),
        # chunks of new prompt tokens on a long context
        dict(name="chunk_bf16", op="attend", batch=2, new_lo=512, new_hi=1024, past_lo=8192, past_hi=16384, hq=32, hkv=8,
             dim=128, page=16, type="bf16", store="16bit", mean=False, window=0, sinks=0, mix=9),
        # the same against a quantised cache, odd lengths
        dict(name="chunk_int8_fp16", op="attend", batch=3, new_lo=333, new_hi=1500, past_lo=1001, past_hi=8000, hq=32,
             hkv=8, dim=128, page=64, type="fp16", store="int8", mean=True, window=0, sinks=0, mix=10),
        # a whole prompt under a sliding window with sinks, small heads
        dict(name="prompt_window_fp16_d64", op="attend", batch=1, new_lo=8192, new_hi=8192, past_lo=0, past_hi=0, hq=16,
             hkv=4, dim=64, page=128, type="fp16", store="16bit", mean=False, window=1024, sinks=4, mix=11),
        # continuous batching: single tokens and chunks of other sequences in one call
        dict(name="mixed_batch_bf16", op="attend", batch=16, new_lo=1, new_hi=256, past_lo=0, past_hi=3800, hq=16, hkv=4,
             dim=128, page=16, type="bf16", store="16bit", mean=False, window=0, sinks=0, mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend"])
    c = dict(op=op, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), type=rng.choice(["fp16", "bf16"]),
             store=rng.choice(["16bit", "int8"]), mix=rng.randrange(1 << 30))
    c["mean"] = c["store"] == "int8" and rng.random() < 0.5
    c["hkv"] = rng.choice([1, 2, 3, 4, 8, 16])
    if op != "attend":
        c["new_hi"] = _log(rng, 1, 9000)
        c["new_lo"] = rng.randint(1, c["new_hi"])
        c["batch"] = max(1, min(_log(rng, 1, 128), 60_000_000 // (c["new_hi"] * c["hkv"] * c["dim"])))
        c["past_hi"] = _log(rng, 1, 4000)
        c["past_lo"] = rng.randint(0, c["past_hi"])
        return c
    c["hq"] = c["hkv"] * rng.choice([1, 2, 4, 5, 8] if c["hkv"] < 16 else [1, 2])
    form = rng.choice(["token", "few", "chunk"])
    if form == "token":
        c["new_lo"] = c["new_hi"] = 1
    elif form == "few":
        c["new_lo"], c["new_hi"] = 1, rng.randint(2, 8)
    else:
        c["new_hi"] = _log(rng, 9, 2048)
        c["new_lo"] = rng.randint(1, c["new_hi"])
    c["past_hi"] = _log(rng, 1, 32000 if form != "chunk" else 9000)
    c["past_lo"] = rng.randint(0, c["past_hi"])
    # scores of the plain form (padded) and the cache both stay below the largest listed case's
    top = c["past_hi"] + c["new_hi"]
    most = min(800_000_000 // (c["hq"] * c["new_hi"] * top), 500_000_000 // (c["hkv"] * c["dim"] * top))
    c["batch"] = max(1, min(_log(rng, 1, 96), most))
    c["window"], c["sinks"] = (_log(rng, 16, 4096), rng.choice([0, 1, 4, 64])) if rng.random() < 0.4 else (0, 0)
    return c


def _lengths(case):
    """(new tokens, tokens held after them) of every sequence: the case's own mix, spread over its ranges."""
    r = random.Random(case["mix"])

    def spread(lo, hi, n):
        got = [hi, lo][: min(n, 2) if lo != hi else 0]
        while len(got) < n:
            got.append(_log(r, max(lo, 1), max(hi, 1)) if hi else 0)
        r.shuffle(got)
        return got

    new = spread(case["new_lo"], case["new_hi"], case["batch"])
    past = spread(case["past_lo"], case["past_hi"], case["batch"])
    return new, [a + b for a, b in zip(new, past)]


def _visible(case):
    """(query, key) pairs that the mask leaves per query head, and the keys that some query of each sequence sees."""
    new, lens = _lengths(case)
    w, s = case["window"], case["sinks"]
    pairs = keys = 0
    for n, total in zip(new, lens):
        first = total - n  # position of the first query
        if not w:
            pairs += n * first + n * (n + 1) // 2
            keys += total
            continue
        for p in range(first, total):
            lo = max(0, p + 1 - w)
            pairs += p + 1 - lo + min(s, lo)
        lo = max(0, first + 1 - w)
        keys += total - lo + min(s, lo)
    return pairs, keys


def work(case):
    new, lens = _lengths(case)
    n, row = sum(new), case["hkv"] * case["dim"]
    held = row * 2 if case["store"] == "16bit" else row + 4 * case["hkv"]  # bytes of one token's keys (or values)
    if case["op"] == "write":
        if case["store"] == "16bit":
            return {"bytes": 2 * n * (row * 2 + held), "flops": 0}
        # read, written, read back, written out; a maximum and a product per value on the way in, a product out
        return {"bytes": 2 * n * (row * 2 + held) * 2, "flops": 2 * n * row * 5}
    if case["op"] == "read":
        return {"bytes": 2 * n * (row * 2 + held), "flops": 2 * n * row if case["store"] == "int8" else 0}
    pairs, keys = _visible(case)
    return {"bytes": 2 * keys * held + 2 * n * case["hq"] * case["dim"] * 2, "flops": 4 * case["dim"] * case["hq"] * pairs}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 17)
    dt = TYPES[case["type"]]
    new, lens = _lengths(case)
    page, hkv, dim, batch = case["page"], case["hkv"], case["dim"], case["batch"]
    need = [-(-n // page) for n in lens]
    width, pages = max(need) + 1, sum(need) + 3
    # pages of a running server: taken in no order, entries behind a sequence's last page unused
    order = torch.randperm(pages, generator=gen, device=DEV)[: sum(need)].to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
    valid = torch.arange(width, device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[valid] = order

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)

    centre = randn(hkv, dim) * 2 if case["mean"] else None  # channel offsets of keys
    s = dict(case=case, page_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
             cu=torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32), max_new=max(new), total=sum(new),
             k_mean=centre, page=page)
    full = (pages, hkv, page, dim)
    if case["store"] == "int8":
        s["k_cache"] = torch.randint(-127, 128, full, generator=gen, device=DEV, dtype=torch.int8)
        s["v_cache"] = torch.randint(-127, 128, full, generator=gen, device=DEV, dtype=torch.int8)
        # absolute maxima of rows of about dim normal values
        s["k_scale"] = (2.0 + 1.5 * torch.rand(full[:3], generator=gen, device=DEV)) / 127
        s["v_scale"] = (2.0 + 1.5 * torch.rand(full[:3], generator=gen, device=DEV)) / 127
        if case["op"] == "attend":  # scores as spread as those of normal keys and queries
            s["k_scale"] *= 0.6
    else:
        s["k_cache"], s["v_cache"] = randn(*full).to(dt), randn(*full).to(dt)
        s["k_scale"] = s["v_scale"] = None
    if case["op"] == "write":
        k = randn(sum(new), hkv, dim)
        s["k"], s["v"] = (k if centre is None else k + centre).to(dt), randn(sum(new), hkv, dim).to(dt)
    if case["op"] == "attend":
        s["q"] = randn(sum(new), case["hq"], dim).to(dt)
    s["dtype"] = dt
    if own:
        import tribench_b200 as tb
        s["cache"] = tb.PagedKVCache(s["k_cache"], s["v_cache"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                     k_mean=centre, dtype=dt)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        import tribench_b200 as tb
        cache, table, lens, cu = s["cache"], s["page_table"], s["seq_lens"], s["cu"]
        if case["op"] == "write":
            cache.append(s["k"], s["v"], table, lens, cu)
            if case["store"] == "16bit":
                return s["k_cache"], s["v_cache"]
            return *cache.gather(table, lens, cu, total=s["total"]), s["k_scale"], s["v_scale"]
        if case["op"] == "read":
            return cache.gather(table, lens, cu, total=s["total"])
        return tb.run_paged_attn(s["q"], cache, table, lens, cu, max_seqlen_q=s["max_new"],
                                 window=case["window"] or None, sinks=case["sinks"])
    if case["op"] == "write":
        _write(s)
        if case["store"] == "16bit":
            return s["k_cache"], s["v_cache"]
        return *_read(s), s["k_scale"], s["v_scale"]
    if case["op"] == "read":
        return _read(s)
    return _attend(s)


def _places(s):
    """Page and row of every new token."""
    cu, lens = s["cu"].long(), s["seq_lens"].long()
    t = torch.arange(s["total"], device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    p = lens[b] - (cu[b + 1] - cu[b]) + t - cu[b]
    return s["page_table"].long()[b, p // s["page"]], p % s["page"]


def _quantised(x):
    top = x.abs().amax(-1, keepdim=True)
    code = torch.where(top > 0, torch.round(x * 127.0 / top), torch.zeros_like(x))
    return code.to(torch.int8), (top / 127.0)[..., 0]


def _write(s):
    page, row = _places(s)
    if s["k_scale"] is None:
        s["k_cache"][page, :, row] = s["k"]
        s["v_cache"][page, :, row] = s["v"]
        return
    k = s["k"].float()
    if s["k_mean"] is not None:
        k = k - s["k_mean"]
    s["k_cache"][page, :, row], s["k_scale"][page, :, row] = _quantised(k)
    s["v_cache"][page, :, row], s["v_scale"][page, :, row] = _quantised(s["v"].float())


def _values(s, page, row):
    """Keys and values of the given places in 32 bits."""
    k, v = s["k_cache"][page, :, row].float(), s["v_cache"][page, :, row].float()
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][page, :, row][..., None], v * s["v_scale"][page, :, row][..., None]
        if s["k_mean"] is not None:
            k = k + s["k_mean"]
    return k, v


def _read(s):
    k, v = _values(s, *_places(s))
    return k.to(s["dtype"]), v.to(s["dtype"])


def _attend(s):
    case, cu, lens = s["case"], s["cu"].long(), s["seq_lens"].long()
    batch, hkv, dim, g = case["batch"], case["hkv"], case["dim"], case["hq"] // case["hkv"]
    new, keys = s["max_new"], (s["page_table"].shape[1] - 1) * s["page"]
    j = torch.arange(keys, device=DEV)
    held = j[None] < lens[:, None]  # [batch, keys]
    page = torch.where(held, s["page_table"].long()[:, j // s["page"]], 0)
    k, v = _values(s, page, (j % s["page"]).expand(batch, keys))  # [batch, keys, hkv, dim]
    i = torch.arange(new, device=DEV)
    n = cu[1:] - cu[:-1]
    q = s["q"][(cu[:-1, None] + i).clamp(max=s["total"] - 1)].float()  # [batch, new, hq, dim]
    q = q.view(batch, new, hkv, g, dim).permute(0, 2, 3, 1, 4).reshape(batch, hkv, g * new, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(dim ** -0.5).view(batch, hkv, g, new, keys)
    p = (lens - n)[:, None] + i  # [batch, new]: position of each query
    seen = held[:, None, :] & (j <= p[..., None])
    if case["window"]:
        seen &= (j > p[..., None] - case["window"]) | (j < case["sinks"])
    seen = seen[:, None, None]
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top.isfinite(), top, torch.zeros_like(top))).exp_()
    total = scores.sum(-1, keepdim=True)
    o = torch.matmul(scores.view(batch, hkv, g * new, keys), v.transpose(1, 2)).view(batch, hkv, g, new, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(batch, new, hkv * g, dim)
    return o[i[None] < n[:, None]].to(s["dtype"])


# ------------------------------------------------------------------ 64 bits, sequence by sequence
def exact(case, seed):
    s = prepare(case, seed)
    new, lens = _lengths(case)
    table = s["page_table"].cpu()
    mean = 0.0 if s["k_mean"] is None else s["k_mean"].double()
    page = s["page"]

    def where(b, lo, hi):
        p = torch.arange(lo, hi)
        return table[b, p // page].long().to(DEV), (p % page).to(DEV)

    def held(b, lo, hi):
        at, row = where(b, lo, hi)
        k, v = s["k_cache"][at, :, row].double(), s["v_cache"][at, :, row].double()
        if s["k_scale"] is None:
            return k, v
        return (k * s["k_scale"][at, :, row].double().unsqueeze(-1) + mean,
                v * s["v_scale"][at, :, row].double().unsqueeze(-1))

    if case["op"] == "read":
        got = [held(b, lens[b] - new[b], lens[b]) for b in range(case["batch"])]
        return torch.cat([k for k, _ in got]), torch.cat([v for _, v in got])
    if case["op"] == "write":
        at = [where(b, lens[b] - new[b], lens[b]) for b in range(case["batch"])]
        at, row = torch.cat([a for a, _ in at]), torch.cat([r for _, r in at])
        if case["store"] == "16bit":
            k, v = s["k_cache"].double(), s["v_cache"].double()
            k[at, :, row], v[at, :, row] = s["k"].double(), s["v"].double()
            return k, v
        back = []
        for x, off, scale in ((s["k"].double() - mean, mean, s["k_scale"].double()),
                              (s["v"].double(), 0.0, s["v_scale"].double())):
            top = x.abs().max(dim=-1).values
            code = torch.round(x * (127 / top.clamp(min=1e-300)).unsqueeze(-1))
            scale[at, :, row] = top / 127
            back.append((code * (top / 127).unsqueeze(-1) + off, scale))
        return back[0][0], back[1][0], back[0][1], back[1][1]
    g, out, start = case["hq"] // case["hkv"], [], 0
    for b in range(case["batch"]):
        k, v = held(b, 0, lens[b])
        k, v = k.transpose(0, 1), v.transpose(0, 1)  # [hkv, keys, dim]
        key = torch.arange(lens[b], device=DEV)
        for lo in range(0, new[b], 512):
            hi = min(new[b], lo + 512)
            q = s["q"][start + lo:start + hi].double().view(hi - lo, case["hkv"], g, case["dim"])
            q = q.permute(1, 2, 0, 3).reshape(case["hkv"], g * (hi - lo), case["dim"])
            pos = torch.arange(lens[b] - new[b] + lo, lens[b] - new[b] + hi, device=DEV).repeat(g)[:, None]
            see = key[None] <= pos
            if case["window"]:
                see = see & ((key[None] > pos - case["window"]) | (key[None] < case["sinks"]))
            e = (q @ k.transpose(1, 2)) / case["dim"] ** 0.5
            e = torch.softmax(e.masked_fill(~see, float("-inf")), dim=-1)
            o = (e @ v).view(case["hkv"], g, hi - lo, case["dim"]).permute(2, 0, 1, 3)
            out.append(o.reshape(hi - lo, case["hq"], case["dim"]))
        start += new[b]
    return torch.cat(out)
