"""Cases of the operators that check drafted tokens over the paged 8-bit KV cache:
the trees of drafts (ancestor masks and positions from parent rows), attention of
a tree over the cache, verification against the target's probabilities from given
random numbers, and keeping the accepted path (its rows moved together in every
layer's cache, the pages behind it given back).

Every case is one step of a batch of requests that hold `context` cached tokens
and bring a tree of `nodes` rows, row 0 being the token that is certain and the
others drafts; `mix` seeds the lengths and the trees, so that they belong to the case.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"


CASES = [
    # One step of 64 requests after 512-token prompts, a tree of 26 rows each (the batch-decoding configuration).
    dict(name="tree_64x26", op="tree", requests=64, nodes=(26, 26), fan=3, context=(512, 767), mix=1),
    # Many drafts of unlike size, up to the largest tree that a request may bring.
    dict(name="tree_ragged_40", op="tree", requests=40, nodes=(1, 1024), fan=0, context=(0, 4000), mix=2),
    # The smallest call: one request with a short cache, a token and seven drafts.
    dict(name="attend_tree_1", op="attend", requests=1, nodes=(8, 8), fan=2, context=(200, 200), page=64, kv_heads=4,
         group=8, dim=64, rope=True, mix=3),
    # The attention of the 64-request step.
    dict(name="attend_tree_64x26", op="attend", requests=64, nodes=(26, 26), fan=3, context=(512, 767), page=64,
         kv_heads=4, group=8, dim=64, rope=True, mix=4),
    # Few requests with long unlike caches and wide trees.
    dict(name="attend_tree_long_6", op="attend", requests=6, nodes=(40, 40), fan=4, context=(9000, 100000), page=128,
         kv_heads=8, group=8, dim=128, rope=True, mix=5),
    # Trees of unlike size, no head sharing, an odd head size, no rotation.
    dict(name="attend_tree_odd_19", op="attend", requests=19, nodes=(1, 200), fan=0, context=(100, 5000), page=32,
         kv_heads=12, group=1, dim=96, rope=False, mix=6),
    # One request, four drafts in a row that a lookup proposed (no probabilities of their own).
    dict(name="verify_chain_1", op="verify", requests=1, nodes=(5, 5), fan=1, vocab=32000, probs=False, greedy=0.0, mix=7),
    # The 64-request step's trees, drawn from a drafting model's probabilities.
    dict(name="verify_tree_64x26", op="verify", requests=64, nodes=(26, 26), fan=3, vocab=32000, probs=True, greedy=0.0,
         mix=8),
    # A ragged batch, a third of it greedy, some without any row, a large odd vocabulary.
    dict(name="verify_ragged_200", op="verify", requests=200, nodes=(0, 12), fan=2, vocab=100003, probs=False, greedy=0.33,
         mix=9),
    # Keeping the accepted paths of the 64-request step, all 22 layers.
    dict(name="keep_64x26", op="keep", requests=64, nodes=(26, 26), fan=3, context=(512, 767), page=64, kv_heads=4, dim=64,
         layers=22, mix=10),
    # Wide heads and small pages, which most paths cross.
    dict(name="keep_ragged_37", op="keep", requests=37, nodes=(0, 150), fan=0, context=(0, 900), page=16, kv_heads=8,
         dim=128, layers=4, mix=11),
    # Very many requests of a small model.
    dict(name="keep_small_2000", op="keep", requests=2000, nodes=(1, 9), fan=1, context=(0, 300), page=16, kv_heads=1,
         dim=32, layers=2, mix=12),
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
    op = rng.choice(["tree", "attend", "attend", "verify", "verify", "keep"])
    mix, fan = rng.randrange(1 << 30), rng.choice([0, 0, 1, 2, 3, 5])
    if op == "tree":
        hi = _log(rng, 1, 1024)
        most = max(1, min(512, 40_000_000 // (hi * hi)))
        return _plain(dict(op=op, requests=_log(rng, 1, most), nodes=(rng.choice([0, 1, hi]), hi), fan=fan,
                           context=(0, _log(rng, 1, 4000)), mix=mix))
    page = rng.choice([16, 32, 64, 128])
    if op == "attend":
        heads = dict(kv_heads=rng.choice([1, 2, 4, 5, 8, 12]), group=rng.choice([1, 2, 3, 4, 7, 8, 16]),
                     dim=rng.choice([32, 64, 64, 96, 128, 128]), rope=rng.random() < 0.75)
        hi, context = _log(rng, 1, 200), _log(rng, 1, 60000)
        row = heads["kv_heads"] * heads["dim"]
        scores = hi * heads["group"] * heads["kv_heads"] * (context + hi)
        while scores > 700_000_000:
            hi = hi // 2 + 1
            scores = hi * heads["group"] * heads["kv_heads"] * (context + hi)
        most = max(1, min(96, 300_000_000 // (context * row), 1_000_000_000 // scores))
        return _plain(dict(op=op, requests=_log(rng, 1, most), nodes=(rng.choice([1, hi]), hi), fan=fan,
                           context=(context // 3, context), page=page, mix=mix, **heads))
    if op == "verify":
        hi, vocab, probs = _log(rng, 1, 40), _log(rng, 50, 150000), rng.random() < 0.5
        most = max(1, min(256, 50_000_000 // (hi * vocab)))
        return _plain(dict(op=op, requests=_log(rng, 1, most), nodes=(rng.choice([0, 1, hi]), hi), fan=fan, vocab=vocab,
                           probs=probs, greedy=rng.choice([0.0, 0.0, 0.3, 1.0]), mix=mix))
    heads = dict(kv_heads=rng.choice([1, 2, 4, 5, 8, 12]), dim=rng.choice([32, 64, 64, 96, 128]))
    hi, layers = _log(rng, 1, 200), _log(rng, 1, 40)
    most = max(1, min(500, 60_000_000 // (layers * heads["kv_heads"] * heads["dim"] * (hi + page))))
    return _plain(dict(op=op, requests=_log(rng, 1, most), nodes=(rng.choice([0, 1, hi]), hi), fan=fan,
                       context=(0, _log(rng, 1, 900)), page=page, layers=layers, mix=mix, **heads))


def trees_of(case, seed=0):
    """(context, parents of each request's rows); their sizes are the same for every seed.  fan 1: a chain; more: that
    many children a row, level by level; 0: any earlier row, near ones more often."""
    sizes, rng = random.Random(case["mix"]), random.Random(case["mix"] + seed)
    fan, context, trees = case["fan"], [], []
    for r in range(case["requests"]):
        n = max(r == 0, _log(sizes, case["nodes_lo"], case["nodes_hi"]))  # one row at least
        context.append(_log(rng, case["context_lo"], case["context_hi"]) if "context_lo" in case else 0)
        trees.append([-1 if t == 0 else (t - 1) // fan if fan else t - 1 - int((t - 1) * rng.random() ** 3)
                      for t in range(n)])
    return context, trees


def _pages(n, page):
    return -(-n // page)


def _depths(parents):
    """Rows on the way to each row, itself among them."""
    out = []
    for p in parents:
        out.append(1 if p < 0 else out[p] + 1)
    return out


def _path(parents, end):
    out = []
    while end >= 0:
        out.append(end)
        end = parents[end]
    return out[::-1]


def _ends(case):
    """A request's last accepted row in the cases that keep a path (the same for every seed)."""
    rng = random.Random(case["mix"] + 1)
    return [rng.randrange(len(p)) if p else -1 for p in trees_of(case)[1]]


def work(case):
    context, trees = trees_of(case)
    new = [len(p) for p in trees]
    tokens, requests, most = sum(new), len(new), max(1, max(new))
    if case["op"] == "tree":
        return {"bytes": 4 * (tokens + 2 * requests + tokens + tokens * _pages(most, 32)), "flops": 0}
    if case["op"] == "verify":
        # The rows of a path: the first and, as an estimate, a draft and a half behind it where there are as many; the
        # last one's draft probabilities.
        rows = sum(min(max(_depths(p)), 2.5) for p in trees if p)
        bytes_ = 4 * case["vocab"] * (rows + (sum(1 for p in trees if p) if case["probs"] else 0))
        return {"bytes": int(bytes_) + 4 * (3 * tokens + 5 * requests + 2 * requests * most), "flops": int(4 * rows * case["vocab"])}
    page, width = case["page"], case["kv_heads"] * case["dim"]
    if case["op"] == "keep":
        paths = [_path(p, e) for p, e in zip(trees, _ends(case))]
        moved = sum(sum(1 for i, j in enumerate(path) if i != j) for path in paths)
        values = 2 * case["layers"] * _keep_pool(case) * page * width
        # the moved rows read and written, the cache read back as values, the requests' lengths
        return {"bytes": 2 * 2 * moved * width * case["layers"] + 5 * values + 4 * 4 * requests + 4 * sum(map(len, paths)), "flops": 0}
    heads = case["kv_heads"] * case["group"]
    keys = sum(c + n for c, n in zip(context, new))
    held = sum(_pages(c + n, page) for c, n in zip(context, new))
    pairs = sum(n * c + sum(_depths(p)) for c, n, p in zip(context, new, trees))
    table = 2 * 4 * tokens * (case["dim"] // 2) if case["rope"] else 0
    return {"bytes": 2 * keys * width + 8 * held * case["kv_heads"] + 4 * held + 2 * 4 * tokens * heads * case["dim"] + table +
            4 * tokens * (1 + _pages(most, 32)), "flops": 4 * pairs * heads * case["dim"]}


# ------------------------------------------------------------------ inputs
def _keep_pool(case):
    """Pages of a pool in the cases that keep a path: the requests' last part-filled ones and those behind."""
    context, trees = trees_of(case)
    page = case["page"]
    return sum(_pages(c + len(p), page) - c // page for c, p in zip(context, trees)) + 3


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


def _masks(trees, words):
    """[tokens, words] of each row's ancestors and itself, as bits."""
    out = []
    for parents in trees:
        sets = []
        for t, p in enumerate(parents):
            sets.append((sets[p] if p >= 0 else 0) | 1 << t)
        out += [[((m >> 32 * w & 0xffffffff) ^ 0x80000000) - 0x80000000 for w in range(words)] for m in sets]
    return _int(out).reshape(-1, words)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    context, trees = trees_of(case, seed if case["op"] == "tree" else 0)  # (the lengths that the others hold are the case's)
    new = [len(p) for p in trees]
    tokens, requests, most = sum(new), len(new), max(1, max(new))
    depth = max((max(_depths(p)) for p in trees if p), default=1)
    state = dict(case=case, tokens=tokens, most=most, depth=depth, context=_int(context), new=_int(new),
                 lengths=_int([c + n for c, n in zip(context, new)]), token_offsets=_offsets(new),
                 parents=_int([x for p in trees for x in p]))
    if case["op"] == "tree":
        state.update(table=torch.zeros((requests, 1), dtype=torch.int32, device=DEVICE),
                     page_offsets=_offsets([1] * requests))
        return state
    if case["op"] == "verify":
        vocab = case["vocab"]
        state.update(table=torch.zeros((requests, 1), dtype=torch.int32, device=DEVICE),
                     page_offsets=_offsets([1] * requests))
        state["children"] = max((max(p.count(t) for t in set(p)) for p in trees if p), default=1)
        # A target and a drafting model that mostly agree.  (Small vocabularies are flatter.)
        spread = 1.6 * math.log(vocab) ** 0.5
        logits = torch.randn((tokens, vocab), generator=gen, device=DEVICE).mul_(spread)
        drafted = torch.randn((tokens, vocab), generator=gen, device=DEVICE).add_(logits)
        row = [0] * tokens
        rank, at = [0] * tokens, 0
        for p in trees:
            seen = {}
            for t, x in enumerate(p):
                row[at + t] = at + max(x, 0)
                rank[at + t] = seen[x] = seen.get(x, -1) + 1
            at += len(p)
        row, rank = _int(row).long(), _int(rank).long()
        state["probs"] = None
        if tokens == 0:
            ids = _int([])
        elif case["probs"]:
            probs = torch.softmax(drafted, dim=-1)
            state["probs"] = probs
            # Each child is drawn from its parent's row: the largest of p / (exponential noise).
            noise = torch.empty_like(probs).exponential_(generator=gen)
            ids = (probs[row] / noise).argmax(dim=-1).to(torch.int32)
        else:  # the drafter's best tokens, in order
            best = drafted.topk(min(state["children"], vocab), dim=-1).indices
            ids = best[row, rank.clamp(max=best.shape[1] - 1)].to(torch.int32)
        uniform = lambda n: torch.rand(n, generator=gen, device=DEVICE)  # noqa: E731
        temperature = 0.6 + 0.6 * uniform(requests)
        temperature[uniform(requests) < case["greedy"]] = 0.0
        state.update(logits=logits, ids=ids, accept=uniform(tokens), sample=uniform(requests), temperature=temperature)
        return state
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    after = [_pages(c + n, page) for c, n in zip(context, new)]
    if case["op"] == "keep":
        # Of a request's pages only those that the step wrote to are in the pool; the others are not looked at.
        pool, layers = _keep_pool(case), case["layers"]
        order = torch.randperm(pool, generator=gen, device=DEVICE).to(torch.int32).cpu()
        table = torch.full((requests, max(after) + 1), -1, dtype=torch.int32)
        at = 0
        for s, (c, e) in enumerate(zip(context, after)):
            first = c // page
            table[s, first:e] = order[at:at + e - first]
            at += e - first
        paths = [_path(p, e) for p, e in zip(trees, _ends(case))]
        held = sum(after)
        state.update(table=table.to(DEVICE), page_offsets=_offsets(after), kept=_int([len(p) for p in paths]),
                     path=_int([p + [-1] * (most - len(p)) for p in paths]), taken=_int([held]),
                     free=torch.arange(held + 64, device=DEVICE, dtype=torch.int32),
                     dropped=_pages(most, page) + 1)
        shape = (layers, pool, kv, page, dim)
        scale = 0.02 + 0.04 * torch.rand((2, layers, pool, kv), generator=gen, device=DEVICE)
    else:
        heads, width = kv * case["group"], kv * dim
        qkv = torch.randn((tokens, heads * dim + 2 * width), generator=gen, device=DEVICE)
        held, pool = sum(after), sum(after) + 3
        order = torch.randperm(pool, generator=gen, device=DEVICE).to(torch.int32).cpu()
        table = torch.full((requests, max(after) + 2), -1, dtype=torch.int32)
        at = 0
        for s, e in enumerate(after):
            table[s, :e] = order[at:at + e]
            at += e
        masks = _masks(trees, _pages(most, 32))
        positions = [c + d - 1 for c, p in zip(context, trees) for d in _depths(p)]
        state.update(q=qkv[:, :heads * dim], positions=_int(positions), masks=masks, table=table.to(DEVICE),
                     page_offsets=_offsets(after), keys=max(c + n for c, n in zip(context, new)),
                     rope=_rope(max(positions) + 1, dim) if case["rope"] else None)
        shape = (pool, kv, page, dim)
        scale = 0.02 + 0.02 * torch.rand((2, pool, kv), generator=gen, device=DEVICE)
    state.update(k_codes=_codes(gen, shape), v_codes=_codes(gen, shape), k_scale=scale[0].contiguous(),
                 v_scale=scale[1].contiguous())
    return state


# ------------------------------------------------------------- plain forms
def _owner(s):
    """The request of each row and the row's number in it."""
    requests, tokens = s["new"].numel(), s["tokens"]
    owner = torch.repeat_interleave(torch.arange(requests, device=DEVICE), s["new"].long(), output_size=tokens)
    return owner, torch.arange(tokens, device=DEVICE) - s["token_offsets"].long()[owner]


def _side_by_side(s, values, fill):
    """[requests, most] of a value a row."""
    out = torch.full((s["new"].numel(), s["most"]), fill, dtype=torch.long, device=DEVICE)
    out[_owner(s)] = values.long()
    return out


def _plain_tree(s):
    requests, most = s["new"].numel(), s["most"]
    parents = _side_by_side(s, s["parents"], -1)
    # Who sees whom: itself and its parent, then everybody that these see, and so on.
    seen = torch.eye(most, device=DEVICE).expand(requests, most, most).clone()
    at = parents.clamp(min=0)[..., None]
    seen.scatter_(2, at, torch.maximum(seen.gather(2, at), (parents >= 0)[..., None].float()))
    for _ in range(max(1, s["depth"] - 1).bit_length()):
        seen = torch.bmm(seen, seen).clamp_(max=1)
    owner, t = _owner(s)
    words = _pages(most, 32)
    rows = torch.nn.functional.pad(seen[owner, t], (0, 32 * words - most)).to(torch.int64).reshape(-1, words, 32)
    masks = (rows << torch.arange(32, device=DEVICE)).sum(dim=-1)
    masks = torch.where(masks >= 1 << 31, masks - (1 << 32), masks)
    positions = s["context"].long()[owner] + rows.sum(dim=(1, 2)) - 1
    return {"positions": positions.to(torch.int32), "masks": masks.to(torch.int32)}


def _turn(x, cos, sin):
    """Rotates the pairs (i, i + dim / 2) of x [..., heads, dim] by its rows of the tables."""
    a, b = x.chunk(2, dim=-1)
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_attend(s):
    case = s["case"]
    page, kv, group, dim = case["page"], case["kv_heads"], case["group"], case["dim"]
    requests, tokens, most, keys = case["requests"], s["tokens"], s["most"], s["keys"]
    q = s["q"].reshape(tokens, kv * group, dim)
    if s["rope"] is not None:
        q = _turn(q, *(t[s["positions"].long()] for t in s["rope"]))
    # Requests side by side, padded to the largest tree and the longest cache.
    owner, t = _owner(s)
    rows = torch.zeros((requests, most, kv * group, dim), device=DEVICE)
    rows[owner, t] = q
    rows = rows.reshape(requests, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(requests, kv, group * most, dim)
    pages = _pages(keys, page)
    table = s["table"][:, :pages].long().clamp(min=0)

    def values(codes, scale):
        x = codes[table] * scale[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(requests, kv, pages * page, dim)

    scores = torch.matmul(rows, values(s["k_codes"], s["k_scale"]).transpose(2, 3)).mul_(dim ** -0.5)
    scores = scores.reshape(requests, kv, group, most, pages * page)
    bits = s["masks"].long()[..., None] >> torch.arange(32, device=DEVICE) & 1
    seen = torch.zeros((requests, most, bits.shape[1] * 32), dtype=torch.bool, device=DEVICE)
    seen[owner, t] = bits.reshape(tokens, -1).bool()
    key = torch.arange(pages * page, device=DEVICE)
    drafted = key - s["context"].long()[:, None]  # the key's number among the request's new rows
    inside = (drafted >= 0) & (drafted < most) & (key < s["lengths"].long()[:, None])
    tree = seen.gather(2, drafted.clamp(0, most - 1)[:, None].expand(requests, most, pages * page))
    visible = (drafted < 0)[:, None] | (inside[:, None] & tree)
    scores.masked_fill_(~visible[:, None, None], float("-inf"))
    scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    scores.div_(scores.sum(dim=-1, keepdim=True))
    out = torch.matmul(scores.reshape(requests, kv, group * most, pages * page), values(s["v_codes"], s["v_scale"]))
    out = out.reshape(requests, kv, group, most, dim).permute(0, 3, 1, 2, 4)
    return out[owner, t].reshape(tokens, kv * group * dim)


def _plain_verify(s):
    """All requests a level at a time, a child at a time, in 64 bits (a draw is a comparison with a long sum)."""
    requests, most, vocab = s["new"].numel(), s["most"], s["case"]["vocab"]
    every = torch.arange(requests, device=DEVICE)
    parents, ids = _side_by_side(s, s["parents"], -2), _side_by_side(s, s["ids"], 0)
    accept = torch.zeros((requests, most), dtype=torch.float64, device=DEVICE)
    accept[_owner(s)] = s["accept"].double()
    starts = s["token_offsets"].long()[:-1]
    path = torch.full((requests, most), -1, dtype=torch.long, device=DEVICE)
    tokens = torch.full_like(path, -1)
    kept = torch.zeros(requests, dtype=torch.long, device=DEVICE)
    last = torch.full_like(kept, -1)
    node, walks = torch.zeros_like(kept), s["new"] > 0
    heat = s["temperature"].double()[:, None]
    for level in range(s["depth"]):
        path[:, level] = torch.where(walks, node, -1)
        row = (starts + node).clamp(max=max(0, s["tokens"] - 1))
        x = s["logits"][row].double()
        top = x.amax(dim=-1, keepdim=True)
        p = torch.where(x == top, 1.0, ((x - top) / torch.where(heat > 0, heat, 1.0)).exp())
        best = torch.zeros_like(p).scatter_(1, x.argmax(dim=-1, keepdim=True), 1.0)
        p = torch.where(heat > 0, p / p.sum(dim=-1, keepdim=True), best)
        child = parents == node[:, None]
        order = child.cumsum(dim=-1)
        found, target = torch.full_like(node, -1), p
        for k in range(s["children"]):
            this = child & (order == k + 1)
            there = this.any(dim=-1) & (found < 0) & walks
            c = this.to(torch.int8).argmax(dim=-1)
            token = ids[every, c][:, None]
            one = torch.zeros_like(p).scatter_(1, token, 1.0)
            q = one if s["probs"] is None else s["probs"][row].double()
            taken = there & (accept[every, c] * q.gather(1, token)[:, 0] < p.gather(1, token)[:, 0])
            found = torch.where(taken, c, found)
            left = (p - q).clamp_(min=0)
            mass = left.sum(dim=-1, keepdim=True)
            left = torch.where(mass > 0, left / mass, target)
            p = torch.where((there & ~taken)[:, None], left, p)
        upto = p.cumsum(dim=-1)
        drawn = (upto <= s["sample"].double()[:, None] * upto[:, -1:]).sum(dim=-1).clamp(max=vocab - 1)
        ends = walks & (found < 0)
        last = torch.where(ends, drawn, last)
        kept = kept + walks
        tokens[:, level] = torch.where(walks, torch.where(ends, drawn, ids[every, found.clamp(min=0)]), -1)
        walks, node = walks & ~ends, found.clamp(min=0)
    return {n: v.to(torch.int32) for n, v in dict(path=path, tokens=tokens, kept=kept, next=last).items()}


def _moved(codes, scale, table, context, path, rows, page):
    """Moves rows `path` of each request together in one layer's codes [pages, kv, page, dim], in place."""
    requests, most = path.shape
    to = context[:, None] + torch.arange(most, device=DEVICE)
    source = context[:, None] + path
    moves = rows & (source != to)
    every = torch.arange(requests, device=DEVICE)[:, None]
    from_page, to_page = (table[every, torch.where(moves, p, 0) // page].clamp(min=0) for p in (source, to))
    kept_from, kept_to = from_page[moves], to_page[moves]
    from_row, to_row = (source % page)[moves], (to % page)[moves]
    # (64 bits: a code next to a half is one or the other.)
    x, x_scale = codes[kept_from, :, from_row].double(), scale[kept_from].double()
    need = (x.abs().amax(dim=-1) * x_scale / torch.full_like(x_scale, 127)).float()
    need = torch.where((kept_from == kept_to)[:, None], 0.0, need)
    grown = scale.scatter_reduce(0, kept_to[:, None].expand(need.shape), need, "amax")
    # A grown page's rows are rounded to its new scale: all those that it keeps.
    ratio = scale.double() / grown.double()
    old = torch.round(codes * ratio[:, :, None, None]).to(torch.int8)
    column = torch.arange(page, device=DEVICE)
    kept_rows = torch.zeros((codes.shape[0], page), dtype=torch.bool, device=DEVICE)
    end = context + rows.sum(dim=-1)  # the request's length now
    pages = table.shape[1]
    held = (torch.arange(pages, device=DEVICE)[:, None] * page + column)[None] < end[:, None, None]
    kept_rows[table[table >= 0].long()] = held[table >= 0]
    codes.copy_(torch.where(kept_rows[:, None, :, None], old, codes))
    codes[kept_to, :, to_row] = torch.round(x * (x_scale / grown[kept_to].double())[..., None]).to(torch.int8)
    scale.copy_(grown)


def _plain_keep(s):
    page = s["case"]["page"]
    context, lengths, kept = s["context"].long(), s["lengths"].long(), s["kept"].long()
    rows = torch.arange(s["most"], device=DEVICE)[None] < kept[:, None]
    table = s["table"].long()
    # The layers are like more pages of one pool.
    layers, pool = s["k_codes"].shape[:2]
    shift = torch.arange(layers, device=DEVICE)[:, None, None] * pool
    tables = torch.where(table >= 0, table + shift, -1).reshape(-1, table.shape[1])
    for name in ("k", "v"):
        _moved(s[name + "_codes"].flatten(0, 1), s[name + "_scale"].flatten(0, 1), tables, context.repeat(layers),
               s["path"].long().repeat(layers, 1), rows.repeat(layers, 1), page)
    left = torch.minimum((context + kept).clamp(min=0), lengths)
    before, after = (lengths + page - 1) // page, (left + page - 1) // page
    freed = before - after
    upto = freed.cumsum(0)
    column = torch.arange(s["dropped"], device=DEVICE)
    drops = column < freed[:, None]
    source = table.gather(1, (after[:, None] + column).clamp(max=table.shape[1] - 1))
    place = (s["taken"].long() - upto)[:, None] + column  # each request's pages below those of the one before
    free = s["free"]
    free[place[drops]] = source[drops].to(torch.int32)
    return dict(_read(s), free=free, lengths=left.to(torch.int32), taken=(s["taken"].long() - upto[-1]).to(torch.int32))


def _read(s):
    """The caches as their readers see them."""
    return {"k": s["k_codes"] * s["k_scale"][..., None, None], "k_scale": s["k_scale"],
            "v": s["v_codes"] * s["v_scale"][..., None, None], "v_scale": s["v_scale"]}


# ---------------------------------------------------------------- one pass
def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"tree": _plain_tree, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[op](s)
    import leaf_b200 as lq

    if "plan" not in s:  # the step's plan, which all layers share
        s["plan"] = lq.Kv8Plan(context=s["context"], lengths=s["lengths"], token_offsets=s["token_offsets"],
                               page_offsets=s["page_offsets"], table=s["table"], tokens=s["tokens"],
                               max_tokens=s["most"], page=s["case"].get("page"))
    plan = s["plan"]
    if op == "tree":
        tree = s["tree"] = lq.kv8_tree(s["parents"], plan, out=s.get("tree"))  # its buffers are kept from step to step
        return {"positions": tree.positions, "masks": tree.masks}
    if op == "verify":
        v = s["verdict"] = lq.verify_drafts(s["logits"], s["ids"], s["parents"], plan, s["accept"], s["sample"],
                                            s["temperature"], draft_probs=s["probs"], out=s.get("verdict"))
        return {"path": v.path, "tokens": v.tokens, "kept": v.kept, "next": v.next}
    if op == "keep":
        if "layers" not in s:  # the layers' caches live as long as the program
            s["layers"] = lq.Kv8Layers([lq.Kv8Cache(*layer) for layer in zip(s["k_codes"], s["v_codes"], s["k_scale"],
                                                                             s["v_scale"])])
        lq.kv8_compact(s["layers"], plan, s["path"], s["kept"])
        left = s["left"] = lq.kv8_release(plan, s["kept"], s["free"], s["taken"], out=s.get("left"))
        return dict(_read(s), free=s["free"], lengths=left.lengths, taken=left.taken)
    if "cache" not in s:  # a layer's cache, the step's trees and the workspace
        s["cache"] = lq.Kv8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        s["tree"] = lq.Kv8Tree(s["positions"], s["masks"])
        s["workspace"] = lq.Kv8Workspace(s["q"].device)
    return lq.kv8_tree_attention(s["q"], s["cache"], plan, s["tree"], scale=s["case"]["dim"] ** -0.5, rope=s["rope"],
                                 workspace=s["workspace"])


# ------------------------------------------------- the definitions, 64 bits
def _exact_keep(case, s):
    context, trees = trees_of(case)
    page = case["page"]
    table = s["table"].tolist()
    out = {}
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"].double(), s[name + "_scale"].double()
        for r, (c, parents, end) in enumerate(zip(context, trees, _ends(case))):
            path = _path(parents, end)
            for first in range(0, len(path) + c % page, page):  # a page of the kept rows at a time
                inside = [i for i in range(len(path)) if first <= i + c % page < first + page]
                moves = [i for i in inside if path[i] != i]
                if not moves:
                    continue
                p = table[r][(c + inside[0]) // page]
                source = [(table[r][(c + path[i]) // page], (c + path[i]) % page) for i in moves]
                x = torch.stack([codes[:, a, :, b] * scale[:, a, :, None] for a, b in source])  # [moves, layers, kv, dim]
                need = scale[:, p].clone()
                for value, (a, _) in zip(x, source):
                    if a != p:
                        need = torch.maximum(need, (value.abs().amax(dim=-1) / 127).float().double())  # a scale has 32 bits
                if not torch.equal(need, scale[:, p]):
                    stay = (c + inside[-1]) % page + 1
                    codes[:, p, :, :stay] = torch.round(codes[:, p, :, :stay] * (scale[:, p] / need)[..., None, None])
                for i, value in zip(moves, x):
                    codes[:, p, :, (c + i) % page] = torch.round(value / need[..., None])
                scale[:, p] = need
        out[name], out[name + "_scale"] = codes * scale[..., None, None], scale
    return dict(out, free=None, lengths=None, taken=None)


def exact(case, seed):
    if case["op"] in ("tree", "verify"):
        return None
    s = prepare(case, seed)
    context, trees = trees_of(case)
    if case["op"] == "keep":
        return _exact_keep(case, s) if case["requests"] * case["layers"] <= 5000 else None
    page, kv, group, dim = case["page"], case["kv_heads"], case["group"], case["dim"]
    tokens = s["tokens"]
    if sum(len(p) * (c + len(p)) for c, p in zip(context, trees)) * kv * group * dim > 2e12:
        return None
    q = s["q"].reshape(tokens, kv * group, dim).double()
    if s["rope"] is not None:
        half = dim // 2
        cos, sin = (t.double()[s["positions"].long()][:, None] for t in s["rope"])
        q = torch.cat((q[..., :half] * cos - q[..., half:] * sin, q[..., half:] * cos + q[..., :half] * sin), dim=-1)
    out = torch.empty((tokens, kv, group, dim), dtype=torch.float64, device=DEVICE)
    at = 0
    for r, (c, parents) in enumerate(zip(context, trees)):
        n = len(parents)
        if n == 0:
            continue
        held = s["table"][r, :_pages(c + n, page)].long()
        seen = torch.zeros((n, c + n), dtype=torch.bool)
        seen[:, :c] = True
        for t in range(n):
            seen[t, [c + i for i in _path(parents, t)]] = True
        seen = seen.to(DEVICE)
        for h in range(kv):
            k = (s["k_codes"][held, h].double() * s["k_scale"][held, h].double()[:, None, None]).reshape(-1, dim)[:c + n]
            v = (s["v_codes"][held, h].double() * s["v_scale"][held, h].double()[:, None, None]).reshape(-1, dim)[:c + n]
            x = torch.einsum("tgd,kd->tgk", q[at:at + n, h * group:(h + 1) * group], k) / math.sqrt(dim)
            x = torch.where(seen[:, None], x, -math.inf)
            out[at:at + n, h] = torch.einsum("tgk,kd->tgd", torch.softmax(x, dim=-1), v)
        at += n
    return out.reshape(tokens, kv * group * dim)
