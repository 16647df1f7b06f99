"""Cases of the paged KV cache's further operators: appending with the position rotation on the way, a cache held
in 4 bits and attention over it, and attention over the blocks that a cheap score selects.

Sequence b brings n_b new tokens and has L_b in all; its token i stands at position L_b - n_b + i. Query head h reads KV head
h // (heads / kv_heads).

Rotation: pair i of a query or key at position p turns by p * inv_freq[i]; the pairs are (i, i + rot / 2), or (2i, 2i + 1) where
they are interleaved, and the dimensions from rot on stay. What is rotated is rounded to the rows' type, and stored as that.

Four bits: a vector x is held as x_d = scale * r_g * c_d, c whole in [-7, 7], r whole in [0, 255] for each group g of 32 dimensions.
With a = max |x| and a_g that of the group: scale = a / 1785, r_g = ceil(255 a_g / a), c = round(x * 1785 / (a * r_g)), ties to even.
A byte holds c + 8 of dimensions 2i (low) and 2i + 1 (high).

Blocks: a block is one page of a sequence. Its bounds are the least and the greatest value of its keys in each dimension. For a query
token a KV head's complete block scores sum over the head's queries of sum_d max(q_d least_d, q_d greatest_d). A token attends
to `take` blocks (all, where it has no more): the first, the last two, its own among them, and the best of the others."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8, "i4": torch.uint8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}  # the largest code of an 8-bit cache
GROUP, TOP4, RATIO = 32, 7.0, 255.0
FIRST, LAST = 1, 2  # blocks that every token attends to


def listed():
    c = _case
    return [
        # a batch of prompts goes into the cache as it is
        c("append bf16 prompts", "append", "bf16", 8, (1000, 2048), (1000, 2048), 32, 8, 128, "bf16", 64, rot=128),
        # prompts into a 4-bit cache, half of the dimensions rotated, by neighbours
        c("append i4 prompts", "append", "f16", 5, (301, 1500), (301, 4001), 16, 4, 128, "i4", 32, rot=64, interleaved=True),
        # a generation step at far positions into an 8-bit cache: latency
        c("append e4m3 step", "append", "bf16", 64, (1, 1), (1000, 131072), 32, 8, 128, "e4m3", 64, rot=128),
        # a generation step of a big batch over a 4-bit cache
        c("step i4", "paged", "bf16", 64, (1, 1), (1000, 8192), 32, 8, 128, "i4", 64),
        # one user, one very long context
        c("step i4 one long", "paged", "bf16", 1, (1, 1), (100001, 100001), 32, 4, 128, "i4", 128),
        # a few short chats on a small model: latency
        c("step i4 small", "paged", "f16", 4, (1, 1), (100, 900), 8, 2, 64, "i4", 16),
        # chunked prefill of long prompts over a 4-bit cache (the largest)
        c("chunk i4", "paged", "bf16", 2, (1024, 2048), (6000, 16000), 32, 8, 128, "i4", 64),
        # a generation step over long contexts, 2048 of up to 32768 keys
        c("blocks bf16", "blocks", "bf16", 32, (1, 1), (8000, 32768), 32, 8, 128, "bf16", 64, take=32),
        # the same out of a 4-bit cache
        c("blocks i4", "blocks", "bf16", 32, (1, 1), (8000, 32768), 32, 8, 128, "i4", 64, take=32),
        # one very long context
        c("blocks f16 one long", "blocks", "f16", 1, (1, 1), (131071, 131071), 32, 4, 128, "f16", 32, take=64),
        # short turns over long documents
        c("blocks e4m3 turns", "blocks", "bf16", 3, (17, 150), (5000, 20000), 16, 4, 64, "e4m3", 64, take=16),
        # fp32 callers
        c("blocks f32", "blocks", "f32", 4, (1, 9), (700, 5001), 8, 4, 80, "f32", 16, take=24),
    ]


def _case(name, op, kind, batch, new, keys, heads, kv_heads, dim, cache, page, rot=0, interleaved=False, take=0):
    """new, keys: the fewest and the most of the batch."""
    return {"name": name, "op": op, "type": kind, "batch": batch, "new_lo": new[0], "new_hi": new[1], "keys_lo": keys[0], "keys_hi": keys[1],
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page, "rot": rot, "interleaved": interleaved, "take": take}


def draw(rng):
    def between(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["append", "paged", "paged", "blocks", "blocks"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":  # codes are made from 16-bit rows
        cache = rng.choice([kind, kind, "i4", "i4", "e4m3", "i8"]) if kind != "f32" else kind
    else:
        cache = "i4" if op == "paged" else rng.choice([kind, kind, "i4", "e4m3", "i8"])
    dim = rng.choice([64, 96, 128, 128]) if cache == "i4" else rng.choice([64, 80, 96, 128, 128])
    batch = between(1, 64)
    rot = take = 0
    if op == "append":
        most = 1 if rng.random() < 0.4 else between(1, 2048)
        longest = max(most, between(16, 200000))
        rot = rng.choice([dim, dim, dim // 2, 16])
    elif op == "paged":
        most = 1 if rng.random() < 0.5 else between(1, 2048)
        longest = max(most, between(16, 20000))
    else:
        most = 1 if rng.random() < 0.6 else between(1, 200)
        longest = max(most, between(64, 60000))
        take = between(FIRST + LAST + 1, 64)
    new = (1 if rng.random() < 0.5 else most, most)
    keys = (max(most, between(1, longest)), longest)
    c = _case("", op, kind, batch, new, keys, heads, kv_heads, dim, cache, page, rot, rng.random() < 0.4, take)
    del c["name"]
    while c["batch"] > 1 and _dear(c):
        c["batch"] = max(1, c["batch"] // 2)
    while _dear(c):
        c["new_hi"] = max(1, c["new_hi"] * 2 // 3)
        c["new_lo"] = min(c["new_lo"], c["new_hi"])
        c["keys_hi"] = max(c["new_hi"], c["keys_hi"] * 9 // 10)
        c["keys_lo"] = min(max(c["keys_lo"], c["new_hi"]), c["keys_hi"])
        c["take"] = max(min(c["take"], FIRST + LAST + 1), c["take"] * 9 // 10)
    return c


def _dear(c):
    """Dearer than the largest listed cases, in the plain form's memory, in bytes or in products of the type."""
    w = work(c)
    return _plain_values(c) > 3e9 or w["bytes"] > 1e9 or w["flops"] > (5e10 if c["type"] == "f32" else 7e11)


def _plain_values(c):
    n, keys, width = c["new_hi"], c["keys_hi"], c["kv_heads"] * c["dim"]
    if c["op"] == "append":
        return 4 * c["batch"] * n * (2 * width + c["heads"] * c["dim"])
    if c["op"] == "paged":
        return c["batch"] * (c["heads"] * n * keys + 2 * keys * width)
    held = c["batch"] * keys * width  # in the cache
    return held + 4 * c["batch"] * n * min(c["take"] * c["page"], keys + c["page"]) * width


def _spread(count, lo, hi, step):
    """`count` whole numbers from lo to hi, both of them among them where count > 1."""
    if count == 1:
        return [hi]
    inner = [lo + int((hi - lo + 1) * ((k * step) % 1.0)) for k in range(1, count - 1)]
    return [lo] + inner + [hi]


def _lengths(c):
    new = _spread(c["batch"], c["new_lo"], c["new_hi"], 0.6180339887)
    keys = _spread(c["batch"], c["keys_lo"], c["keys_hi"], 0.4142135623)
    return new, [max(n, k) for n, k in zip(new, keys)]


def _stored(c):
    """Bytes of one vector in the cache."""
    D = c["dim"]
    if c["cache"] == "i4":
        return D // 2 + D // GROUP + 4
    return D * BYTES[c["cache"]] + (4 if c["cache"] in TOP else 0)


def work(case):
    c = case
    new, keys = _lengths(c)
    H, D, heads, page = c["kv_heads"], c["dim"], c["heads"], c["page"]
    tokens, b, stored = sum(new), BYTES[c["type"]], _stored(c)
    rows = 2 * tokens * heads * D * b  # queries and what comes of them
    if c["op"] == "append":
        return {"bytes": rows + 4 * tokens * H * (D * b + stored), "flops": 3 * tokens * (heads + H) * c["rot"]}
    if c["op"] == "paged":
        pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(new, keys))
        return {"bytes": rows + 2 * sum(keys) * H * stored, "flops": 4 * D * heads * pairs}
    most = c["take"]
    bound = 2 * D * (4 if c["type"] == "f32" else 2)
    scored = read = made = flops = 0
    for n, k in zip(new, keys):
        blocks = -(-k // page)
        made += k // page - (k - n) // page
        others = max(0, blocks - FIRST - LAST) if blocks > most else 0
        scored += others
        read += min(blocks, most)  # new tokens of a sequence may agree
        flops += n * (4 * D * H * others + 4 * D * heads * min(k, most * page))
    return {"bytes": rows + H * (scored * bound + made * (page * stored + bound) + read * page * 2 * stored + tokens * most * 4), "flops": flops}


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[c["type"]]

    def values(*shape, by=1.0):
        return torch.randn(shape, device="cuda", generator=g).mul_(by).to(kind)

    def starts(counts):
        return torch.tensor([0] + counts, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()

    new, keys = _lengths(c)
    total, H, D, page = sum(new), c["kv_heads"], c["dim"], c["page"]
    s = {"case": c, "cu": starts(new), "most_new": max(new), "lens": torch.tensor(keys, dtype=torch.int32).cuda(), "q": values(total, c["heads"], D, by=1.5)}
    if c["op"] == "append":  # keys with a few strong channels, as after a projection
        s["k"] = values(total, H, D).mul_(values(1, H, D).abs_().add_(0.5))
        s["v"] = values(total, H, D)
        s["inv_freq"] = (500000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])).float().cuda()
    # A pool whose pages lie in any order, with some to spare, all holding what earlier sequences left there. What only
    # appends is given the pages that it writes to.
    slots = [-(-k // page) for k in keys]
    from_ = [(k - n) // page if c["op"] == "append" else 0 for n, k in zip(new, keys)]
    need = [n - f for n, f in zip(slots, from_)]
    pages = sum(need) + 7
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(c["batch"], max(slots), dtype=torch.int32, device="cuda")
    rows = torch.repeat_interleave(torch.arange(c["batch"]), torch.tensor(need)).cuda()
    cols = torch.cat([torch.arange(f, n) for f, n in zip(from_, slots)]).cuda()
    table[rows, cols] = order[: sum(need)]
    s["table"] = table
    for name in ("k", "v"):
        scale = group = None
        if c["cache"] == "i4":
            codes = torch.randint(1, 16, (pages, H, page, D // 2), device="cuda", generator=g, dtype=torch.uint8)
            codes += torch.randint(1, 16, codes.shape, device="cuda", generator=g, dtype=torch.uint8) << 4
            scale = torch.rand(pages, H, page, device="cuda", generator=g).add_(0.5).mul_(2.0 / 1785)
            group = torch.zeros(pages, H, page, 4 * -(-D // 128), device="cuda", dtype=torch.uint8)
            group[..., : D // GROUP] = torch.randint(120, 256, (pages, H, page, D // GROUP), device="cuda", generator=g, dtype=torch.uint8)
            group[..., 0] = 255
        elif c["cache"] in TOP:
            codes = torch.randint(-112, 113, (pages, H, page, D), device="cuda", generator=g, dtype=torch.int8)
            if c["cache"] == "e4m3":
                codes = (codes.half() * 2.0).to(TYPES["e4m3"])
            scale = torch.rand(pages, H, page, device="cuda", generator=g).add_(0.5).mul_(2.0 / TOP[c["cache"]])
        else:
            codes = torch.randn(pages, H, page, D, device="cuda", generator=g).to(TYPES[c["cache"]])
            if c["op"] == "blocks":  # neighbours have something in common
                codes += torch.randn(pages, H, 1, D, device="cuda", generator=g).to(codes.dtype)
        s |= {name + "_pages": codes, name + "_scale": scale, name + "_group": group}
    if c["op"] == "blocks":
        s["bounds"] = torch.zeros(pages, H, 2, D, dtype=kind, device="cuda")
        for first in range(0, pages, 4096):
            at = slice(first, first + 4096)
            x = _values(s["k_pages"][at], *(None if t is None else t[at] for t in (s["k_scale"], s["k_group"])))
            s["bounds"][at, :, 0], s["bounds"][at, :, 1] = x.amin(2), x.amax(2)
        # the blocks that the new tokens complete have none yet
        for b, (n, k) in enumerate(zip(new, keys)):
            s["bounds"][table[b, (k - n) // page: k // page].long()] = 0
    return s


def run(state):
    op = state["case"]["op"]
    return _append(state) if op == "append" else _paged(state) if op == "paged" else _blocks(state)


def _append(s):
    """Queries rotated, keys and values in the cache, and read back from there."""
    c, k_pages, v_pages = s["case"], s["k_pages"], s["v_pages"]
    scales = {name: s[name] for name in ("k_scale", "v_scale", "k_group", "v_group")}
    if own:
        capi = _capi()
        q, k, v = (torch.empty_like(s[name]) for name in ("q", "k", "v"))
        where = s["cu"], s["table"], s["lens"]
        capi.kv_pages_append_rope_dev(s["k"], s["v"], k_pages, v_pages, *where, s["inv_freq"], c["interleaved"], Q=s["q"], Q_out=q, **scales)
        capi.kv_pages_read_dev(k_pages, v_pages, k, v, *where, **scales)
        return q, k, v
    b, position = _positions(s)
    where, slot = s["table"][b, position // c["page"]].long(), position % c["page"]
    angle = position[:, None].double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q, k = (_rotated(s[name].float(), cos, sin, c["interleaved"]).to(s[name].dtype) for name in ("q", "k"))
    _store(k.float(), k_pages, s["k_scale"], s["k_group"], where, slot)
    _store(s["v"].float(), v_pages, s["v_scale"], s["v_group"], where, slot)
    k, v = (_values(*(None if t is None else t[where, :, slot] for t in (s[name + "_pages"], s[name + "_scale"], s[name + "_group"]))) for name in ("k", "v"))
    return q, k.to(s["k"].dtype), v.to(s["v"].dtype)


def _paged(s):
    if own:
        o = torch.empty_like(s["q"])
        scales = {name: s[name] for name in ("k_scale", "v_scale", "k_group", "v_group")}
        _capi().attn_paged_dev(s["q"], s["k_pages"], s["v_pages"], o, s["cu"], s["table"], s["lens"], s["most_new"], **scales)
        return o
    at, there = _padded(s["cu"], s["most_new"])
    table = s["table"].long()
    k, v = (_values(*(None if t is None else t[table] for t in (s[x + "_pages"], s[x + "_scale"], s[x + "_group"]))).transpose(1, 2).flatten(2, 3) for x in ("k", "v"))
    q = s["q"].float()[at]
    B, n, heads, D = q.shape
    H, L = k.shape[1], k.shape[2]
    q = (q / math.sqrt(D)).view(B, n, H, -1, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    z = torch.matmul(q, k.transpose(2, 3)).view(B, H, -1, n, L)
    last = (s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long())[:, None] + torch.arange(n, device=q.device)
    seen = torch.arange(L, device=q.device) <= last[..., None].clamp(max=s["lens"].long()[:, None, None] - 1)
    o = torch.matmul(_weights(z, seen[:, None, None]).flatten(2, 3), v)
    return o.view(B, H, -1, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, heads, D)[there].to(s["q"].dtype)


def _blocks(s):
    """As after an append: bounds of the blocks that are complete now, the blocks of each new token, attention to them."""
    c = s["case"]
    page, take = c["page"], c["take"]
    where = s["cu"], s["table"], s["lens"]
    if own:
        capi = _capi()
        o = torch.empty_like(s["q"])
        blocks = torch.empty(s["q"].shape[0], c["kv_heads"], take, dtype=torch.int32, device="cuda")
        capi.kv_blocks_bounds_dev(s["k_pages"], s["bounds"], *where, k_scale=s["k_scale"], k_group=s["k_group"])
        capi.kv_blocks_select_dev(s["q"], s["bounds"], blocks, *where, page, keep_first=FIRST, keep_last=LAST)
        capi.attn_blocks_dev(s["q"], s["k_pages"], s["v_pages"], o, blocks, *where, k_scale=s["k_scale"], v_scale=s["v_scale"], k_group=s["k_group"], v_group=s["v_group"])
        return o, blocks, s["bounds"]
    table, lens = s["table"].long(), s["lens"].long()
    # bounds
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    most = (s["most_new"] + page - 1) // page + 1
    slot = ((lens - new) // page)[:, None] + torch.arange(most, device="cuda")
    made = table.gather(1, slot.clamp(max=table.shape[1] - 1))[slot < (lens // page)[:, None]]
    x = _values(*(None if t is None else t[made] for t in (s["k_pages"], s["k_scale"], s["k_group"])))
    s["bounds"][made] = torch.stack([x.amin(2), x.amax(2)], 2).to(s["bounds"].dtype)
    # scores, in 64 bits for those next to the last one taken
    at, there = _padded(s["cu"], s["most_new"])
    B, n, P, H, D, take_ = len(lens), s["most_new"], table.shape[1], c["kv_heads"], c["dim"], min(take, table.shape[1])
    q = s["q"].double()[at].view(B, n, H, -1, D)
    q = torch.cat([q.clamp(max=0).sum(3), q.clamp(min=0).sum(3)], -1).transpose(1, 2)
    score = torch.matmul(q, s["bounds"][table].double().permute(0, 2, 3, 4, 1).flatten(2, 3))
    last = ((lens - new)[:, None] + torch.arange(n, device="cuda")) // page  # the block of the token itself
    j = torch.arange(P, device="cuda")
    score = torch.where((j < FIRST) | (j > last[:, None, :, None] - LAST), torch.inf, score)
    score = torch.where(j > last[:, None, :, None], -torch.inf, score)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :take_]
    best = torch.where(best <= last[:, None, :, None], best, P).sort(-1)[0].transpose(1, 2)[there]  # [tokens, H, take_]
    blocks = torch.full((best.shape[0], H, take), -1, dtype=torch.int32, device="cuda")
    blocks[..., :take_] = torch.where(best < P, best, -1)
    # attention
    b, position = _positions(s)
    pages = table[b[:, None, None], best.clamp(max=P - 1)]
    head = torch.arange(H, device="cuda")[None, :, None]
    k, v = (_values(*(None if t is None else t[pages, head] for t in (s[x + "_pages"], s[x + "_scale"], s[x + "_group"]))).flatten(2, 3) for x in ("k", "v"))
    seen = (best[..., None] * page + torch.arange(page, device="cuda") <= position[:, None, None, None]).flatten(2)[:, :, None]
    q = s["q"].float().view(len(b), H, -1, D) / math.sqrt(D)
    o = torch.matmul(_weights(torch.matmul(q, k.transpose(2, 3)), seen), v)
    return o.reshape(s["q"].shape).to(s["q"].dtype), blocks, s["bounds"]


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


def _positions(s):
    """Sequence and position of each packed token."""
    token = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(s["cu"][1:].contiguous(), token, right=True)
    return b, s["lens"][b].long() - s["cu"][b + 1] + token


def _rotated(x, cos, sin, interleaved):
    half = cos.shape[-1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _weights(z, seen):
    z = z.masked_fill(~seen, float("-inf"))
    z = z.sub_(z.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = z.sum(-1, keepdim=True)
    return z / torch.where(total > 0, total, 1.0)


def _values(codes, scale, group):
    """What pages hold, in 32 bits."""
    if group is not None:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
        codes = codes * group[..., : codes.shape[-1] // GROUP].float().repeat_interleave(GROUP, -1)
    return codes.float() if scale is None else codes.float() * scale[..., None]


def _store(x, pages, scale, group, where, slot):
    """x in fp32 into its places; codes in 64 bits, for the values next to a border between two of them."""
    if scale is None:
        pages[where, :, slot] = x.to(pages.dtype)
        return
    most = x.abs().amax(-1, keepdim=True)
    some = torch.where(most > 0, most, 1.0).double()
    if group is not None:
        each = x.abs().unflatten(-1, (-1, GROUP)).amax(-1)
        ratio = (RATIO * each.double() / some).ceil()
        spread = torch.where(ratio > 0, ratio, 1.0).repeat_interleave(GROUP, -1)
        codes = (x.double() * (TOP4 * RATIO) / (some * spread)).round().to(torch.int16) + 8
        pages[where, :, slot] = (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8)
        scale[where, :, slot] = (most / (TOP4 * RATIO))[..., 0]
        group[where, :, slot] = torch.nn.functional.pad(ratio, (0, group.shape[-1] - ratio.shape[-1])).to(torch.uint8)
        return
    top = TOP["i8" if pages.dtype == torch.int8 else "e4m3"]
    t = x.double() * top / some
    if pages.dtype == torch.int8:
        codes = t.round().to(torch.int8)
    else:
        step = torch.ldexp(torch.ones_like(t), torch.frexp(t)[1].clamp(min=-5) - 4)
        codes = ((t / step).round() * step).float().to(pages.dtype)
    pages[where, :, slot] = codes
    scale[where, :, slot] = (most / top)[..., 0]


def exact(case, seed):
    """From the definition, sequence by sequence and head by head."""
    c = case
    new, keys = _lengths(c)
    s = prepare(case, seed)
    if c["op"] == "append":
        return _exact_append(s, new, keys)
    H, D, G = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    o = torch.zeros(sum(new), c["heads"], D, dtype=torch.float64, device="cuda")
    if c["op"] == "blocks":
        if sum(new) * H > 4000:
            return None
        return _exact_blocks(s, new, keys, o)
    first = 0
    for b, (n, L) in enumerate(zip(new, keys)):
        k, v = (_exact_tokens(s, x, b, L) for x in ("k", "v"))
        past = torch.ones(n, L, dtype=torch.bool, device="cuda").tril(L - n)
        for h in range(c["heads"]):
            z = s["q"][first:first + n, h].double() @ k[:, h // G].T / D ** 0.5
            o[first:first + n, h] = torch.softmax(torch.where(past, z, -torch.inf), 1) @ v[:, h // G]
        first += n
    return o


def _exact_pages(s, name, pages):
    """The tokens of these pages, [pages * page, kv_heads, D]."""
    x = s[name + "_pages"][pages]
    if s[name + "_group"] is not None:
        low = x.remainder(16).double() - 8
        high = x.div(16, rounding_mode="floor").double() - 8
        x = torch.empty(*x.shape[:-1], 2 * x.shape[-1], dtype=torch.float64, device=x.device)
        x[..., 0::2], x[..., 1::2] = low, high
        for g in range(x.shape[-1] // GROUP):
            x[..., g * GROUP:(g + 1) * GROUP] *= s[name + "_group"][pages][..., g, None].double()
    x = x.double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][pages].double().unsqueeze(-1)
    return x.permute(0, 2, 1, 3).flatten(0, 1)


def _exact_tokens(s, name, b, L):
    return _exact_pages(s, name, s["table"][b, : -(-L // s["case"]["page"])].long())[:L]


def _exact_blocks(s, new, keys, o):
    c = s["case"]
    H, D, G, page, take = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"], c["page"], c["take"]
    bounds = s["bounds"].double()
    token = 0
    for b, (n, L) in enumerate(zip(new, keys)):
        at = s["table"][b].long()
        for j in range((L - n) // page, L // page):
            x = _exact_pages(s, "k", at[j:j + 1]).float()
            bounds[at[j], :, 0] = x.min(0).values.to(s["q"].dtype).double()
            bounds[at[j], :, 1] = x.max(0).values.to(s["q"].dtype).double()
        for i in range(n):
            p = L - n + i
            mine = p // page
            for h in range(H):
                q = s["q"][token, h * G:(h + 1) * G].double()
                chosen = torch.arange(mine + 1, device="cuda")
                if mine + 1 > take:
                    low, high = bounds[at[:mine + 1], h].unbind(1)
                    score = torch.maximum(q[:, None] * low, q[:, None] * high).sum((0, 2))
                    inner = score[FIRST:mine + 1 - LAST].sort(descending=True, stable=True).indices[: take - FIRST - LAST] + FIRST
                    chosen = torch.cat([chosen[:FIRST], inner.sort().values, chosen[-LAST:]])
                where = at[chosen]
                here = (chosen[:, None] * page + torch.arange(page, device="cuda")).flatten() <= p
                one = {x + end: None if s[x + end] is None else s[x + end][where, h:h + 1] for x in ("k", "v") for end in ("_pages", "_scale", "_group")}
                every = torch.arange(len(where), device="cuda")
                k, v = (_exact_pages(one, x, every)[here, 0] for x in ("k", "v"))
                o[token, h * G:(h + 1) * G] = torch.softmax(q @ k.T / D ** 0.5, 1) @ v
            token += 1
    return o, None, bounds


def _exact_append(s, new, keys):
    c = s["case"]
    position = torch.cat([torch.arange(k - n, k) for n, k in zip(new, keys)]).cuda()
    turn = torch.polar(torch.ones(len(position), len(s["inv_freq"]), dtype=torch.float64, device="cuda"), torch.outer(position.double(), s["inv_freq"].double()))
    half = len(s["inv_freq"])
    first = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else half)
    out = []
    for name in ("q", "k", "v"):
        x = s[name].double()
        if name != "v":
            z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
            x[..., first], x[..., second] = z.real, z.imag
        if name != "q":
            x = _exact_codes(x.to(s[name].dtype).double(), c["cache"])
        out.append(x)
    return tuple(out)


def _exact_codes(x, cache):
    if cache not in TOP and cache != "i4":
        return x
    most = x.abs().max(-1, keepdim=True).values
    most = torch.where(most > 0, most, torch.ones_like(most))
    if cache == "i4":
        shape = x.shape
        x = x.reshape(*shape[:-1], -1, GROUP)
        most = most[..., None]
        ratio = torch.ceil(RATIO * x.abs().max(-1, keepdim=True).values / most)
        ratio = torch.where(ratio > 0, ratio, 1)
        return (torch.round(x * (TOP4 * RATIO) / (most * ratio)) * ratio * most / (TOP4 * RATIO)).reshape(shape)  # (a tie stays one in this order)
    y = x * TOP[cache] / most
    grid = torch.ones_like(y) if cache == "i8" else 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / grid) * grid * (most / TOP[cache])
