"""Cases of the serving operators: attention over packed prompts, a paged KV cache that is quantised as it is
written, and attention of new tokens over that cache.

Sequence b brings n_b new tokens and has L_b keys in all; its query i stands at position L_b - n_b + i and sees
the keys up to there. Query head h reads KV head h // (heads / kv_heads)."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}  # the largest code of an 8-bit cache


def listed():
    c = _case
    return [
        # long documents of one upload, as one packed prefill (the largest)
        c("packed bf16 long", "packed", "bf16", 2, (5000, 8000), (0, 0), 32, 8, 128),
        # a full prefill batch at the attention block's size: hidden 4096, up to 2048 tokens a sequence
        c("packed f16 batch", "packed", "f16", 4, (1024, 2048), (0, 0), 32, 8, 128),
        # fp32 callers of the dense prefill, with grouped heads
        c("packed f32", "packed", "f32", 3, (101, 901), (0, 0), 16, 4, 64),
        # a handful of short chat turns: latency
        c("packed bf16 short", "packed", "bf16", 5, (1, 60), (0, 0), 8, 2, 64),
        # an ordinary generation step
        c("step bf16", "paged", "bf16", 32, (1, 1), (500, 4096), 32, 8, 128, "bf16", 64),
        # a generation step of a big batch over an 8-bit cache
        c("step e4m3", "paged", "bf16", 64, (1, 1), (1000, 8192), 32, 8, 128, "e4m3", 32),
        # one user, one very long context
        c("step bf16 one long", "paged", "bf16", 1, (1, 1), (100001, 100001), 32, 4, 128, "bf16", 128),
        # the dense decode step's size (8 x 32 heads, 4096 keys) out of pages
        c("step f32", "paged", "f32", 8, (1, 1), (4096, 4096), 32, 32, 128, "f32", 16),
        # chunked prefill mixed with shorter pieces, an odd head size
        c("chunk f16 mixed", "paged", "f16", 6, (1, 700), (1500, 9000), 16, 2, 80, "f16", 16),
        # chunked prefill of long prompts over an 8-bit cache
        c("chunk i8", "paged", "bf16", 2, (1024, 2048), (6000, 16000), 32, 8, 128, "i8", 128),
        # prompts go into the cache and come back out, as when they are moved to another pool
        c("cache e4m3 prompts", "cache", "bf16", 8, (1000, 2048), (1000, 2048), 32, 8, 128, "e4m3", 64),
        # one token a sequence in and out: latency
        c("cache i8 step", "cache", "f16", 16, (1, 1), (1, 1), 32, 8, 128, "i8", 16),
    ]


def _case(name, op, kind, batch, new, keys, heads, kv_heads, dim, cache="", page=0):
    """new, keys: the shortest and the longest of the batch. A packed prompt's keys are its own tokens. For
    "cache", keys counts the tokens read back, the last ones of each sequence, those just written among them."""
    return {"name": name, "op": op, "type": kind, "batch": batch, "new_lo": new[0], "new_hi": new[1], "keys_lo": keys[0], "keys_hi": keys[1],
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page}


def draw(rng):
    def between(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["packed", "packed", "paged", "paged", "paged", "cache"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    cache, page = "", 0
    if op == "packed":
        batch, longest = between(1, 24), between(8, 6000)
        new, keys = (between(1, longest), longest), (0, 0)
    else:
        cache, page = rng.choice([kind, kind, "e4m3", "i8"]), rng.choice([16, 32, 64, 128])
        batch = between(1, 64)
        most = 1 if op == "paged" and rng.random() < 0.5 else between(1, 2048)
        new = (1 if rng.random() < 0.5 else most, most)
        longest = max(most, between(16, 20000 if op == "paged" else 4000))
        keys = (max(most, between(1, longest)), longest)
    c = _case("", op, kind, batch, new, keys, heads, kv_heads, dim, cache, page)
    del c["name"]
    while c["batch"] > 1 and _dear(c):
        c["batch"] = max(1, c["batch"] // 2)
    while _dear(c):
        c["new_hi"] = max(1, c["new_hi"] * 2 // 3)
        c["new_lo"] = min(c["new_lo"], c["new_hi"])
        if op != "packed":
            c["keys_hi"] = max(c["new_hi"], c["keys_hi"] * 9 // 10)
            c["keys_lo"] = min(max(c["keys_lo"], c["new_hi"]), c["keys_hi"])
    return c


def _dear(c):
    """Dearer than the largest listed cases, in the plain form's memory, in bytes or in products of the type."""
    w = work(c)
    return _plain_values(c) > 3e9 or w["bytes"] > 1e9 or w["flops"] > (2e11 if c["type"] == "f32" else 7e11)


def _plain_values(c):
    n, keys = c["new_hi"], c["new_hi"] if c["op"] == "packed" else c["keys_hi"]
    score = 0 if c["op"] == "cache" else c["heads"] * n * keys
    return c["batch"] * (score + 2 * keys * c["kv_heads"] * c["dim"])


def _spread(count, lo, hi, step):
    """`count` whole numbers from lo to hi, both of them among them where count > 1."""
    if count == 1:
        return [hi]
    inner = [lo + int((hi - lo + 1) * ((k * step) % 1.0)) for k in range(1, count - 1)]
    return [lo] + inner + [hi]


def _lengths(c):
    new = _spread(c["batch"], c["new_lo"], c["new_hi"], 0.6180339887)
    if c["op"] == "packed":
        return new, new
    keys = _spread(c["batch"], c["keys_lo"], c["keys_hi"], 0.4142135623)
    return new, [max(n, k) for n, k in zip(new, keys)]


def work(case):
    c = case
    new, keys = _lengths(c)
    width, tokens = c["kv_heads"] * c["dim"], sum(new)
    b = BYTES[c["type"]]
    if c["op"] == "cache":
        stored = width * BYTES[c["cache"]] + (4 * c["kv_heads"] if c["cache"] in TOP else 0)
        held = sum(keys) - tokens  # tokens that were there before and are only read
        return {"bytes": 2 * (tokens * width * b + tokens * stored + held * stored + sum(keys) * width * b), "flops": 0}
    pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(new, keys))
    flops = 4 * c["dim"] * c["heads"] * pairs
    if c["op"] == "packed":
        return {"bytes": b * tokens * (2 * c["heads"] * c["dim"] + 2 * width), "flops": flops}
    stored = width * BYTES[c["cache"]] + (4 * c["kv_heads"] if c["cache"] in TOP else 0)
    return {"bytes": b * tokens * 2 * c["heads"] * c["dim"] + 2 * sum(keys) * stored, "flops": flops}


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[c["type"]]

    def values(*shape, by=1.0):
        return torch.randn(shape, device="cuda", generator=g).mul_(by).to(kind)

    def starts(counts):
        return torch.tensor([0] + counts, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()

    new, keys = _lengths(c)
    total, H, D = sum(new), c["kv_heads"], c["dim"]
    s = {"case": c, "cu": starts(new), "most_new": max(new), "most_keys": max(keys)}
    if c["op"] != "cache":
        s["q"] = values(total, c["heads"], D, by=1.5)
    if c["op"] != "paged":  # keys with a few strong channels, as after a projection
        s["k"] = values(total, H, D).mul_(values(1, H, D).abs_().add_(0.5))
        s["v"] = values(total, H, D)
    if c["op"] == "packed":
        return s
    # a pool whose pages lie in any order, with some to spare, all holding what earlier sequences left there
    page = c["page"]
    need = [-(-k // page) for k in keys]
    pages = sum(need) + 7
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(c["batch"], max(need), dtype=torch.int32, device="cuda")
    rows = torch.repeat_interleave(torch.arange(c["batch"]), torch.tensor(need)).cuda()
    cols = torch.cat([torch.arange(n) for n in need]).cuda()
    table[rows, cols] = order[: sum(need)]
    s |= {"table": table, "lens": torch.tensor(keys, dtype=torch.int32).cuda(), "k_scale": None, "v_scale": None}
    for name in ("k", "v"):
        if c["cache"] in TOP:
            codes = torch.randint(-112, 113, (pages, H, page, D), device="cuda", generator=g, dtype=torch.int8)
            if c["cache"] == "e4m3":
                codes = (codes.half() * 2.0).to(TYPES["e4m3"])
            s[name + "_pages"] = codes
            s[name + "_scale"] = torch.rand(pages, H, page, device="cuda", generator=g).add_(0.5).mul_(2.0 / TOP[c["cache"]])
        else:
            s[name + "_pages"] = torch.randn(pages, H, page, D, device="cuda", generator=g).to(TYPES[c["cache"]])
    if c["op"] == "cache":
        s["cu_read"] = starts(keys)
        s["read"] = sum(keys)
    return s


def run(state):
    op = state["case"]["op"]
    return _packed(state) if op == "packed" else _paged(state) if op == "paged" else _cache(state)


def _packed(s):
    if own:
        o = torch.empty_like(s["q"])
        _capi().attn_packed_dev(s["q"], s["k"], s["v"], o, s["cu"], causal=True)
        return o
    at, there = _padded(s["cu"], s["most_new"])
    q, k, v = (s[name].float()[at] for name in ("q", "k", "v"))
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    return _attention(q, k.transpose(1, 2), v.transpose(1, 2), n, n)[there].to(s["q"].dtype)


def _paged(s):
    if own:
        o = torch.empty_like(s["q"])
        _capi().attn_paged_dev(s["q"], s["k_pages"], s["v_pages"], o, s["cu"], s["table"], s["lens"], s["most_new"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return o
    at, there = _padded(s["cu"], s["most_new"])
    k, v = (_unpaged(s[name + "_pages"], s[name + "_scale"], s["table"]) for name in ("k", "v"))
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    return _attention(s["q"].float()[at], k, v, n, s["lens"].long())[there].to(s["q"].dtype)


def _cache(s):
    k_pages, v_pages, k_scale, v_scale = s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]
    if own:
        capi = _capi()
        k, v = (torch.empty(s["read"], *s["k"].shape[1:], dtype=s["k"].dtype, device="cuda") for _ in range(2))
        capi.kv_pages_append_dev(s["k"], s["v"], k_pages, v_pages, s["cu"], s["table"], s["lens"], k_scale=k_scale, v_scale=v_scale)
        capi.kv_pages_read_dev(k_pages, v_pages, k, v, s["cu_read"], s["table"], s["lens"], k_scale=k_scale, v_scale=v_scale)
        return k, v
    page = k_pages.shape[2]
    where, slot = _places(s["cu"], s["k"].shape[0], s["table"], s["lens"], page)
    for x, pages, scale in ((s["k"], k_pages, k_scale), (s["v"], v_pages, v_scale)):
        if scale is None:
            pages[where, :, slot] = x.to(pages.dtype)
        else:
            codes, step = _quantised(x, pages.dtype)
            pages[where, :, slot] = codes
            scale[where, :, slot] = step
    where, slot = _places(s["cu_read"], s["read"], s["table"], s["lens"], page)
    k, v = (pages[where, :, slot].float() if scale is None else pages[where, :, slot].float() * scale[where, :, slot][..., None]
            for pages, scale in ((k_pages, k_scale), (v_pages, v_scale)))
    return k.to(s["k"].dtype), v.to(s["v"].dtype)


def _capi():
    import sys
    if "attn-cpu_b200" not in sys.path:
        sys.path.insert(0, "attn-cpu_b200")
    from attn_cpu import capi
    return capi


def _padded(cu, most):
    """Row numbers of every sequence's tokens, [batch, most], and which of them are there."""
    at = cu[:-1, None].long() + torch.arange(most, device=cu.device)
    there = at < cu[1:, None]
    return torch.where(there, at, 0), there


def _attention(q, k, v, new, keys):
    """q [B, n, heads, D], k and v [B, kv_heads, L, D], all fp32 -> [B, n, heads, D]."""
    B, n, heads, D = q.shape
    H, L = k.shape[1], k.shape[2]
    G = heads // H
    q = (q * (1.0 / math.sqrt(D))).view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    s = torch.matmul(q, k.transpose(2, 3)).view(B, H, G, n, L)
    j = torch.arange(L, device=q.device)
    last = (keys - new)[:, None] + torch.arange(n, device=q.device)  # the last key that a query sees
    seen = (j <= last[..., None]) & (j < keys[:, None, None])
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, H, G * n, L), v).view(B, H, G, n, D)
    o = o / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, heads, D)


def _unpaged(pages, scale, table):
    """[B, kv_heads, L, D] in fp32, L whole pages."""
    x = pages[table.long()].float()
    if scale is not None:
        x = x * scale[table.long()][..., None]
    B, P, H, page, D = x.shape
    return x.transpose(1, 2).reshape(B, H, P * page, D)


def _places(cu, total, table, lens, page):
    """Page and slot of each packed token: the last ones of their sequences."""
    token = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    position = lens[b] - cu[b + 1] + token
    return table[b, position // page].long(), position % page


def _quantised(x, dtype):
    """Codes and steps; in 64 bits, for the values next to a border between two codes."""
    top = TOP["i8" if dtype == torch.int8 else "e4m3"]
    most = x.abs().amax(-1, keepdim=True)
    t = x.double() * top / torch.where(most > 0, most, 1.0).double()
    if dtype == torch.int8:
        codes = t.round().to(torch.int8)
    else:
        step = torch.ldexp(torch.ones_like(t), torch.frexp(t)[1].clamp(min=-5) - 4)
        codes = ((t / step).round() * step).float().to(dtype)
    return codes, (most.float() / top)[..., 0]


def exact(case, seed):
    """From the definition, sequence by sequence and head by head."""
    c = case
    new, keys = _lengths(c)
    s = prepare(case, seed)
    H, D, G = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    if c["op"] == "cache":
        return _exact_cache(s, new, keys)
    o = torch.zeros(sum(new), c["heads"], D, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, L) in enumerate(zip(new, keys)):
        if c["op"] == "packed":
            k, v = (s[x][first:first + n].double() for x in ("k", "v"))
        else:
            k, v = (_exact_tokens(s, x, b, L) for x in ("k", "v"))
        past = torch.ones(n, L, dtype=torch.bool, device="cuda").tril(L - n)
        for h in range(c["heads"]):
            q = s["q"][first:first + n, h].double()
            z = torch.einsum("id,jd->ij", q, k[:, h // G]) / D ** 0.5
            z = torch.where(past, z, -torch.inf)
            o[first:first + n, h] = torch.einsum("ij,jd->id", torch.softmax(z, 1), v[:, h // G])
        first += n
    return o


def _exact_tokens(s, name, b, L):
    """The first L tokens of sequence b as the pages hold them, [L, kv_heads, D]."""
    pages = s["table"][b, : -(-L // s["case"]["page"])].long()
    x = s[name + "_pages"][pages].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][pages].double().unsqueeze(-1)
    return x.permute(0, 2, 1, 3).flatten(0, 1)[:L]


def _exact_cache(s, new, keys):
    got = {"k": [], "v": []}
    first = 0
    for b, (n, L) in enumerate(zip(new, keys)):
        for name, to in got.items():
            x = s[name][first:first + n].double()
            kind = s["case"]["cache"]
            if kind in TOP:
                most = x.abs().max(-1, keepdim=True).values
                y = x * TOP[kind] / torch.where(most > 0, most, torch.ones_like(most))  # a tie stays one in this order
                if kind == "e4m3":  # 3 bits behind the leading one, from 2^-6 up; the multiples of 2^-9 below that
                    near = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
                    grid = 2.0 ** (near - 3)
                else:
                    grid = torch.ones_like(y)
                x = torch.round(y / grid) * grid * (most / TOP[kind])
            else:
                x = x.to(TYPES[kind]).double()
            to.append(torch.cat([_exact_tokens(s, name, b, L)[: L - n], x]))
        first += n
    return torch.cat(got["k"]), torch.cat(got["v"])
