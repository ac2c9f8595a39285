"""Cases of the paged 8-bit KV cache operators: the step plan (block tables and
slot maps from request lengths), the append that rotates and quantises new keys
and values into the cache, and causal grouped-query attention over it.

Every case is one step of a batch of requests that hold `context` cached tokens
and bring `new` ones; `mix` seeds the lengths, so that they belong to the case.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"


CASES = [
    # One decode step of 64 requests after 512-token prompts: one new token each (the batch-decoding configuration).
    dict(name="plan_decode_64", op="plan", requests=64, new=(1, 1), context=(512, 767), page=64, mix=1),
    # Admission of many requests at once: ragged prompts, some with nothing new, small pages.
    dict(name="plan_ragged_2000", op="plan", requests=2000, new=(0, 1000), context=(0, 4000), page=16, mix=2),
    # The append of that decode step for one layer of the 1.1B shape (4 kv heads of 64).
    dict(name="append_decode_64", op="append", requests=64, new=(1, 1), context=(512, 767), page=64, kv_heads=4,
         group=8, dim=64, rope=True, mix=3),
    # The append of 64 prompts of 512 tokens: the prefill of the same configuration.
    dict(name="append_prompts_64x512", op="append", requests=64, new=(512, 512), context=(0, 0), page=64, kv_heads=4,
         group=8, dim=64, rope=True, mix=4),
    # Chunks of unlike lengths that continue part-filled pages, wide heads, small pages.
    dict(name="append_ragged_37", op="append", requests=37, new=(1, 700), context=(0, 900), page=16, kv_heads=8,
         group=4, dim=128, rope=True, mix=5),
    # The smallest call: one request, one token, a short cache (batch-1 decoding, positions 128..255).
    dict(name="attend_decode_1", op="attend", requests=1, new=(1, 1), context=(200, 200), page=64, kv_heads=4,
         group=8, dim=64, rope=True, mix=6),
    # The attention of the 64-request decode step.
    dict(name="attend_decode_64", op="attend", requests=64, new=(1, 1), context=(512, 767), page=64, kv_heads=4,
         group=8, dim=64, rope=True, mix=7),
    # Few requests with long unlike caches: the work has to be split along the keys.
    dict(name="attend_decode_long", op="attend", requests=6, new=(1, 1), context=(9000, 100000), page=128, kv_heads=8,
         group=8, dim=128, rope=True, mix=8),
    # A few tokens a request (checking drafted tokens), no head sharing, an odd head size, no rotation.
    dict(name="attend_draft_19", op="attend", requests=19, new=(4, 4), context=(100, 5000), page=32, kv_heads=12,
         group=1, dim=96, rope=False, mix=9),
    # The attention of 64 prompts of 512 tokens.
    dict(name="attend_prompts_64x512", op="attend", requests=64, new=(512, 512), context=(0, 0), page=64, kv_heads=4,
         group=8, dim=64, rope=True, mix=10),
    # Chunked prefill: unlike chunks behind unlike cached prefixes, three query heads to a kv head, small pages.
    dict(name="attend_chunks_5", op="attend", requests=5, new=(100, 1500), context=(0, 5000), page=16, kv_heads=8,
         group=3, dim=128, rope=True, mix=11),
    # One long prompt.
    dict(name="attend_prompt_8192", op="attend", requests=1, new=(8192, 8192), context=(0, 0), page=64, kv_heads=4,
         group=8, dim=64, rope=True, mix=12),
]


def _plain(case):
    """A case as plain values: each range as two numbers."""
    out = {}
    for key, value in case.items():
        if isinstance(value, tuple):
            out[key + "_lo"], out[key + "_hi"] = value
        else:
            out[key] = value
    return out


def listed():
    return [_plain(c) for c in CASES]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 2))) - 1)))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    mix = rng.randrange(1 << 30)
    if op == "plan":
        new = rng.choice([(1, 1), (0, _log(rng, 1, 1000))])
        return _plain(dict(op=op, requests=_log(rng, 1, 2000), new=new, context=(1, _log(rng, 1, 4000)), page=page, mix=mix))
    heads = dict(kv_heads=rng.choice([1, 2, 4, 5, 8, 12]), group=rng.choice([1, 2, 3, 4, 7, 8, 16]),
                 dim=rng.choice([32, 64, 64, 96, 128, 128]), rope=rng.random() < 0.75)
    if op == "append":
        hi = rng.choice([1, _log(rng, 1, 700)])
        most = max(1, min(128, 24_000_000 // (2 * hi * heads["kv_heads"] * heads["dim"])))
        return _plain(dict(op=op, requests=_log(rng, 1, most), new=(1, hi), context=(0, _log(rng, 1, 900)), page=page,
                           mix=mix, **heads))
    row = heads["kv_heads"] * heads["dim"]
    if rng.random() < 0.5:  # decode: one or a few tokens, any cache
        hi = rng.choice([1, 1, 2, 4, 9])
        context = _log(rng, 1, 60000)
        rows = hi * heads["group"] * heads["kv_heads"]
        most = max(1, min(96, 200_000_000 // (context * row), 300_000_000 // (context * rows)))
        return _plain(dict(op=op, requests=_log(rng, 1, most), new=(1, hi), context=(context // 3, context), page=page,
                           mix=mix, **heads))
    hi = _log(rng, 10, 4000)
    context = rng.choice([0, _log(rng, 1, 5000)])
    scores = hi * (hi + context) * heads["kv_heads"] * heads["group"]
    most = max(1, min(64, 1_000_000_000 // scores))
    while scores > 1_000_000_000:
        hi, context = hi // 2 + 1, context // 2
        scores = hi * (hi + context) * heads["kv_heads"] * heads["group"]
    return _plain(dict(op=op, requests=_log(rng, 1, most), new=(rng.choice([1, hi]), hi), context=(context // 4, context),
                       page=page, mix=mix, **heads))


def lengths_of(case):
    """(context, new) of every request, the same for every seed."""
    rng = random.Random(case["mix"])
    new, context = [], []
    for _ in range(case["requests"]):
        new.append(_log(rng, case["new_lo"], case["new_hi"]))
        context.append(_log(rng, case["context_lo"], case["context_hi"]))
    return context, new


def _pages(n, page):
    return -(-n // page)


def work(case):
    context, new = lengths_of(case)
    page, tokens, requests = case["page"], sum(new), len(new)
    held = sum(_pages(c + n, page) for c, n in zip(context, new))
    if case["op"] == "plan":
        fresh = held - sum(_pages(c, page) for c in context)
        # lengths in and out, both prefixes, the new table entries (read from the free list, written), position and slot
        return {"bytes": 4 * (2 * requests + 3 * requests + 2 * fresh + 2 * tokens), "flops": 0}
    width = case["kv_heads"] * case["dim"]
    table = 2 * 4 * tokens * (case["dim"] // 2) if case["rope"] else 0
    if case["op"] == "append":
        # the rows in, their codes out, the scales of the touched pages, and the cache read back as values
        touched = sum(_pages(c + n, page) - c // page for c, n in zip(context, new) if n)
        values = 2 * _append_pool(case) * page * width
        return {"bytes": 2 * 4 * tokens * width + 2 * tokens * width + 2 * 8 * touched * case["kv_heads"] + table + 8 * tokens
                + 5 * values, "flops": 6 * tokens * width}
    heads = case["kv_heads"] * case["group"]
    keys = sum(c + n for c, n in zip(context, new))
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(context, new))
    return {"bytes": 2 * keys * width + 8 * held * case["kv_heads"] + 4 * held + 2 * 4 * tokens * heads * case["dim"] + table,
            "flops": 4 * pairs * heads * case["dim"]}


# ------------------------------------------------------------------ inputs
def _append_pool(case):
    """Pages of an append's pool: those that the step touches (the requests' full pages are not needed) and a few more."""
    context, new = lengths_of(case)
    return sum(_pages(c + n, case["page"]) - c // case["page"] for c, n in zip(context, new) if n) + 3


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _offsets(values):
    total, out = 0, [0]
    for v in values:
        total += v
        out.append(total)
    return _int(out)


def _rope(rows, dim):
    """cos and sin of every position, [rows, dim / 2]."""
    rate = 10000.0 ** (-torch.arange(0, dim, 2, device=DEVICE, dtype=torch.float64) / dim)
    angle = torch.arange(rows, device=DEVICE, dtype=torch.float64)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _codes(gen, shape):
    """Codes as rows of normal values give them."""
    x = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float16)
    return x.mul_(38).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    context, new = lengths_of(case)
    page, tokens, requests = case["page"], sum(new), len(new)
    before = [_pages(c, page) for c in context]
    after = [_pages(c + n, page) for c, n in zip(context, new)]
    held = sum(after)
    state = dict(case=case, tokens=tokens, most=max(new), context=_int(context), new=_int(new))
    if case["op"] == "plan":
        # The pool's pages in any order: what the requests hold first, then the free ones.
        shuffled = torch.randperm(held + 64, generator=gen, device=DEVICE).to(torch.int32)
        most = max(after) + 8
        table = torch.full((requests, most), -1, dtype=torch.int32)
        owned, at = shuffled.cpu(), 0
        for s, b in enumerate(before):
            table[s, :b] = owned[at:at + b]
            at += b
        state.update(table=table.to(DEVICE), free=shuffled, taken=_int([at]))
        return state
    kv, dim, group = case["kv_heads"], case["dim"], case["group"]
    heads = kv * group
    qkv = torch.randn((tokens, (heads + 2 * kv) * dim), generator=gen, device=DEVICE)
    # Keys of real models have a few channels that are much larger than the rest.
    loud = 1 + 4 * (torch.rand(kv * dim, generator=gen, device=DEVICE) < 0.05).float()
    qkv[:, heads * dim:(heads + kv) * dim] *= loud
    q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], dim=1)
    positions = [c + t for c, n in zip(context, new) for t in range(n)]
    state.update(q=q, k=k, v=v, positions=_int(positions), token_offsets=_offsets(new),
                 lengths=_int([c + n for c, n in zip(context, new)]), rope=_rope(max(positions) + 1, dim) if case["rope"] else None)
    if case["op"] == "append":
        # Only pages that the step writes: the request's part-filled one and those behind it.
        pool = _append_pool(case)
        order = torch.randperm(pool, generator=gen, device=DEVICE).cpu().tolist()
        slots, at = [], 0
        for c, n in zip(context, new):
            first = c // page
            slots += [order[at + p // page - first] * page + p % page for p in range(c, c + n)]
            if n:
                at += _pages(c + n, page) - first
        state["slots"] = _int(slots)
        # Some part-filled pages hold smaller values than what comes: their scale has to grow.
        scale = 0.02 + 0.06 * torch.rand((2, pool, kv), generator=gen, device=DEVICE)
    else:
        pool = held + 3
        order = torch.randperm(pool, generator=gen, device=DEVICE).to(torch.int32).cpu()
        table = torch.full((requests, max(after) + 2), -1, dtype=torch.int32)
        at = 0
        for s, e in enumerate(after):
            table[s, :e] = order[at:at + e]
            at += e
        state.update(table=table.to(DEVICE), page_offsets=_offsets(after), keys=max(c + n for c, n in zip(context, new)))
        scale = 0.02 + 0.02 * torch.rand((2, pool, kv), generator=gen, device=DEVICE)
    state.update(k_codes=_codes(gen, (pool, kv, page, dim)), v_codes=_codes(gen, (pool, kv, page, dim)),
                 k_scale=scale[0].contiguous(), v_scale=scale[1].contiguous())
    return state


# ------------------------------------------------------------- plain forms
def _turn(x, cos, sin):
    """Rotates the pairs (i, i + dim / 2) of x [..., heads, dim] by its rows of the tables."""
    a, b = x.chunk(2, dim=-1)
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_plan(s):
    page, table, free, taken = s["case"]["page"], s["table"], s["free"], s["taken"]
    context, new, tokens = s["context"].long(), s["new"].long(), s["tokens"]
    most = table.shape[1]
    before, after = (context + page - 1) // page, (context + new + page - 1) // page
    fits = after <= most
    need = torch.where(fits, after - before, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (taken.long() + upto <= free.numel()))
    lengths = torch.where(granted, context + new, context)
    column = torch.arange(most, device=table.device)[None]
    fresh = granted[:, None] & (column >= before[:, None]) & (column < after[:, None])
    source = taken.long() + (upto - need - before)[:, None] + column
    table = torch.where(fresh, free[source.clamp(0, free.numel() - 1)], table)
    zero = torch.zeros(1, dtype=torch.long, device=table.device)
    token_offsets = torch.cat((zero, new.cumsum(0)))
    page_offsets = torch.cat((zero, ((lengths + page - 1) // page).cumsum(0)))
    owner = torch.repeat_interleave(torch.arange(new.numel(), device=table.device), new, output_size=tokens)
    positions = context[owner] + torch.arange(tokens, device=table.device) - token_offsets[owner]
    slots = table[owner, (positions // page).clamp(max=most - 1)] * page + positions % page
    slots = torch.where(granted[owner], slots, -1)
    taken = taken + torch.where(granted & (need > 0), upto, 0).max()
    return {name: x.to(torch.int32) for name, x in dict(
        table=table, lengths=lengths, token_offsets=token_offsets, page_offsets=page_offsets, positions=positions,
        slots=slots, taken=taken).items()}


def _quantise(x, slots, codes, scale):
    """Rows x [tokens, kv, dim] into the slots of codes [pages, kv, page, dim], the pages' scales grown where they must."""
    pages, kv, page, dim = codes.shape
    at, row = slots // page, slots % page
    largest = x.abs().amax(dim=2)
    new_max = torch.zeros_like(scale).scatter_reduce(0, at[:, None].expand(-1, kv), largest, "amax")
    first = torch.full((pages,), page, device=x.device).scatter_reduce(0, at, row, "amin")
    need = (new_max / torch.full_like(new_max, 127)).clamp(min=1e-12)
    grown = torch.where((first > 0)[:, None], torch.maximum(scale, need), need)
    grown = torch.where((first < page)[:, None], grown, scale)
    held = torch.arange(page, device=x.device)[None] < first[:, None]
    old = torch.round(codes * (scale / grown)[:, :, None, None])
    codes = torch.where(held[:, None, :, None], old, codes.float())
    codes[at, :, row] = torch.round(x * (1 / grown)[at][:, :, None]).clamp(-127, 127)
    return codes, grown


def _plain_append(s):
    kv, dim = s["case"]["kv_heads"], s["case"]["dim"]
    k, v = (s[n].reshape(s["tokens"], kv, dim) for n in ("k", "v"))
    slots = s["slots"].long()
    if s["rope"] is not None:
        k = _turn(k, *(t[s["positions"].long()] for t in s["rope"]))
    out = {}
    for name, x in (("k", k), ("v", v)):
        codes, scale = _quantise(x, slots, s[name + "_codes"], s[name + "_scale"])
        out[name], out[name + "_scale"] = codes * scale[:, :, None, None], scale
    return out


def _plain_attend(s):
    case = s["case"]
    page, kv, group, dim = case["page"], case["kv_heads"], case["group"], case["dim"]
    requests, tokens, most, keys = case["requests"], s["tokens"], s["most"], s["keys"]
    q = s["q"].reshape(tokens, kv * group, dim)
    if s["rope"] is not None:
        q = _turn(q, *(t[s["positions"].long()] for t in s["rope"]))
    # Requests side by side, padded to the longest chunk and the longest cache.
    starts = s["token_offsets"].long()
    step = torch.arange(most, device=q.device)[None]
    row = (starts[:-1, None] + step).clamp(max=tokens - 1)
    q = q[row].reshape(requests, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(requests, kv, group * most, dim)
    pages = _pages(keys, page)
    table = s["table"][:, :pages].long().clamp(min=0)

    def values(codes, scale):
        x = codes[table] * scale[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(requests, kv, pages * page, dim)

    scores = torch.matmul(q, values(s["k_codes"], s["k_scale"]).transpose(2, 3)).mul_(dim ** -0.5)
    scores = scores.reshape(requests, kv, group, most, pages * page)
    last = torch.minimum(s["context"].long()[:, None] + step, s["lengths"].long()[:, None] - 1)
    hidden = torch.arange(pages * page, device=q.device) > last[..., None]
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    scores.div_(scores.sum(dim=-1, keepdim=True))
    out = torch.matmul(scores.reshape(requests, kv, group * most, pages * page), values(s["v_codes"], s["v_scale"]))
    out = out.reshape(requests, kv, group, most, dim).permute(0, 3, 1, 2, 4)
    owner = torch.repeat_interleave(torch.arange(requests, device=q.device), s["new"].long(), output_size=tokens)
    return out[owner, torch.arange(tokens, device=q.device) - starts[owner]].reshape(tokens, kv * group * dim)


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[op](state)
    import leaf_b200 as lq

    s = state
    if op == "plan":
        # The plan's buffers are kept from step to step.
        plan = s["plan"] = lq.kv8_plan(s["context"], s["new"], s["table"], s["free"], s["taken"], page=s["case"]["page"],
                                       tokens=s["tokens"], max_tokens=s["most"], out=s.get("plan"))
        return {name: getattr(plan, name) for name in ("table", "lengths", "token_offsets", "page_offsets", "positions",
                                                       "slots", "taken")}
    if "cache" not in s:  # a layer's cache lives as long as the program
        s["cache"] = lq.Kv8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    cache = s["cache"]
    if op == "append":
        lq.kv8_append(s["k"], s["v"], cache, s["slots"], s["positions"], rope=s["rope"])
        # The cache as its readers see it.
        return {"k": cache.k * cache.k_scale[:, :, None, None], "k_scale": cache.k_scale,
                "v": cache.v * cache.v_scale[:, :, None, None], "v_scale": cache.v_scale}
    if "step" not in s:  # the step's plan, which all layers share, and the workspace, which all steps share
        s["step"] = lq.Kv8Plan(context=s["context"], lengths=s["lengths"], token_offsets=s["token_offsets"],
                               page_offsets=s["page_offsets"], table=s["table"], tokens=s["tokens"], max_tokens=s["most"])
        s["workspace"] = lq.Kv8Workspace(s["q"].device)
    return lq.kv8_attention(s["q"], cache, s["step"], scale=s["case"]["dim"] ** -0.5, rope=s["rope"],
                            workspace=s["workspace"])


# ------------------------------------------------- the definitions, 64 bits
def _rotated64(x, positions, rope):
    x = x.double()
    if rope is None:
        return x
    half = x.shape[-1] // 2
    cos, sin = (t.double()[positions][:, None] for t in rope)
    turned = torch.empty_like(x)
    turned[..., :half] = x[..., :half] * cos - x[..., half:] * sin
    turned[..., half:] = x[..., half:] * cos + x[..., :half] * sin
    return turned


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    context, new = lengths_of(case)
    page, kv, group, dim = case["page"], case["kv_heads"], case["group"], case["dim"]
    tokens = sum(new)
    positions = s["positions"].long()
    if case["op"] == "append":
        rows = {"k": _rotated64(s["k"].reshape(tokens, kv, dim), positions, s["rope"]),
                "v": s["v"].reshape(tokens, kv, dim).double()}
        slots = s["slots"].tolist()
        out = {}
        for name, x in rows.items():
            codes, scale = s[name + "_codes"].double(), s[name + "_scale"].double()
            i = 0
            while i < tokens:  # one page of one request at a time
                p, first = divmod(slots[i], page)
                n = 1
                while i + n < tokens and slots[i + n] == slots[i] + n and first + n < page:
                    n += 1
                chunk = x[i:i + n].transpose(0, 1)
                need = torch.clamp(chunk.abs().amax(dim=(1, 2)) / 127, min=1e-12)
                if first:
                    need = torch.maximum(need, scale[p])
                    codes[p, :, :first] = torch.round(codes[p, :, :first] * (scale[p] / need)[:, None, None])
                codes[p, :, first:first + n] = torch.clamp(torch.round(chunk / need[:, None, None]), -127, 127)
                scale[p] = need
                i += n
            out[name], out[name + "_scale"] = codes * scale[:, :, None, None], scale
        return out
    if sum(n * (c + n) for c, n in zip(context, new)) * kv * group * dim > 2e12:
        return None
    q = _rotated64(s["q"].reshape(tokens, kv * group, dim), positions, s["rope"])
    out = torch.empty((tokens, kv, group, dim), dtype=torch.float64, device=DEVICE)
    at = 0
    for r, (c, n) in enumerate(zip(context, new)):
        if n == 0:
            continue
        held = s["table"][r, :_pages(c + n, page)].long()
        for h in range(kv):
            k = (s["k_codes"][held, h].double() * s["k_scale"][held, h].double()[:, None, None]).reshape(-1, dim)[:c + n]
            v = (s["v_codes"][held, h].double() * s["v_scale"][held, h].double()[:, None, None]).reshape(-1, dim)[:c + n]
            rows = q[at:at + n, h * group:(h + 1) * group]
            for b in range(0, n, 2048):
                x = torch.einsum("tgd,kd->tgk", rows[b:b + 2048], k) / math.sqrt(dim)
                seen = torch.arange(c + n, device=DEVICE)[None] <= c + b + torch.arange(x.shape[0], device=DEVICE)[:, None]
                x = torch.where(seen[:, None], x, -math.inf)
                out[at + b:at + b + x.shape[0], h] = torch.einsum("tgk,kd->tgd", torch.softmax(x, dim=-1), v)
        at += n
    return out.reshape(tokens, kv * group * dim)
