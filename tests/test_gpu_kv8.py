"""The paged INT8 cache's operators on the GPU against their definitions in
64-bit floats (oracle/kv8.py).

Tolerances, with u = 2^-24:
* plan: whole numbers, equal.
* append: a scale is a quotient of a rotated value (two products and a sum:
  3 u of the pair's magnitude) by 127, so within 8 u of the exact one; a code
  may differ by one where the exact quotient lies within 127 * 16 u of a half.
* attention: rounding a score of reach R (scale * sum |q||k|) costs at most
  (dim + 16) u R -- each product and each partial sum of the dot, the rotation,
  the scale factors -- and enters the weights of numerator and denominator;
  the exponentials, their sums and the value products add 64 u.  With values
  up to V: |error| <= V * (2 (dim + 16) R + 64) u.  Errors are random, so the
  2-norm of the whole output is held to 1e-5 of its own as well.
"""
import numpy as np
import pytest
import torch

import leaf_b200 as lq
from leaf_b200 import _lib
from oracle import kv8 as ok

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _status_ok():
    return _lib.load().leafq_device_status() == 0


def _rope(rows, rotary):
    rate = 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
    angle = np.arange(rows)[:, None] * rate
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _rope_cuda(rope):
    return None if rope is None else tuple(torch.from_numpy(t).cuda() for t in rope)


# ------------------------------------------------------------------- plan
def _check_plan(context, new, table, free, taken, page, tokens):
    expect = ok.plan(context, new, table, free, taken, page, tokens)
    t = _i32(table)
    got = lq.kv8_plan(_i32(context), _i32(new), t, _i32(free), _i32([taken]), page, tokens)
    torch.cuda.synchronize()
    for name in ("lengths", "token_offsets", "page_offsets", "positions", "slots", "table"):
        assert np.array_equal(getattr(got, name).cpu().numpy(), expect[name]), name
    assert int(got.taken.item()) == expect["taken"]
    return got


def _plan_case(rng, requests, page, longest, most_new):
    context = rng.integers(0, longest + 1, requests)
    new = rng.integers(0, most_new + 1, requests)
    new[rng.random(requests) < 0.2] = 0
    context[rng.random(requests) < 0.2] = 0
    held = [ok.pages_of(int(c), page) for c in context]
    max_pages = max(ok.pages_of(int(c + n), page) for c, n in zip(context, new)) + 1
    order = rng.permutation(sum(held) + int(sum(ok.pages_of(int(n), page) + 1 for n in new)))
    table, at = np.full((requests, max_pages), -1), 0
    for s, b in enumerate(held):
        table[s, :b] = order[at:at + b]
        at += b
    return context, new, table, order, at


@pytest.mark.parametrize("requests", [1, 3, 64, 255, 257, 1025, 2500])
@pytest.mark.parametrize("page,longest,most_new", [(16, 40, 1), (16, 300, 70), (64, 500, 200), (128, 1000, 3)])
def test_plan(cuda_device, requests, page, longest, most_new):
    rng = np.random.default_rng(requests * 1000 + page + most_new)
    context, new, table, order, taken = _plan_case(rng, requests, page, longest, most_new)
    _check_plan(context, new, table, order, taken, page, int(new.sum()))
    _check_plan(context, new, table, order, taken, page, int(new.sum()) + 13)  # rows beyond the last token
    assert _status_ok()


@pytest.mark.parametrize("requests", [5, 300, 1500])
def test_plan_refuses_what_does_not_fit(cuda_device, requests):
    rng = np.random.default_rng(requests)
    context, new, table, order, taken = _plan_case(rng, requests, 16, 200, 90)
    for cut in (0, 1, 7, order.size // 2):  # a pool that ends too early
        _check_plan(context, new, table, order[:taken + cut], taken, 16, int(new.sum()))
    narrow = table[:, :table.shape[1] * 2 // 3].copy()  # rows that end too early
    fits = np.array([ok.pages_of(int(c), 16) <= narrow.shape[1] for c in context])
    _check_plan(context * fits, new, narrow, order, taken, 16, int(new.sum()))
    assert _status_ok()


def test_plan_without_requests_or_tokens(cuda_device):
    table = np.zeros((0, 4), dtype=np.int64)
    _check_plan([], [], table, [3, 1], 0, 32, 0)
    _check_plan([], [], table, [3, 1], 1, 32, 6)
    _check_plan([0, 5, 32], [0, 0, 0], np.array([[-1, -1], [2, -1], [0, -1]]), [], 0, 32, 0)
    assert _status_ok()


def test_plan_reports_negative_lengths_and_too_few_rows(cuda_device):
    got = lq.kv8_plan(_i32([4, -3]), _i32([2, 5]), _i32([[0, 1], [2, 3]]), _i32([4, 5]), _i32([0]), 16, 2)
    torch.cuda.synchronize()
    assert got.slots.tolist() == [4, 5] and got.lengths.tolist() == [6, 0]
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    lq.kv8_plan(_i32([4, 3]), _i32([2, 5]), _i32([[0, 1], [2, 3]]), _i32([4, 5]), _i32([0]), 16, 3)
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    assert _status_ok()


def test_plan_steps_follow_one_another(cuda_device):
    # Ten steps of unlike growth: every step's pages come from where the last stopped.
    rng = np.random.default_rng(5)
    requests, page = 40, 16
    context = np.zeros(requests, dtype=np.int64)
    table, taken = np.full((requests, 40), -1), 0
    free = rng.permutation(requests * 40)
    t, plan = _i32(table), None
    length, count = _i32(context), _i32([0])
    for step in range(10):
        new = rng.integers(0, 40, requests)
        expect = ok.plan(context, new, table, free, taken, page, 2000)
        plan = lq.kv8_plan(length, _i32(new), t, _i32(free), count, page, 2000, out=plan)
        torch.cuda.synchronize()
        assert np.array_equal(t.cpu().numpy(), expect["table"]) and np.array_equal(plan.slots.cpu().numpy(), expect["slots"])
        length.copy_(plan.lengths)
        count.copy_(plan.taken)
        context, table, taken = expect["lengths"], expect["table"], expect["taken"]
        live = expect["slots"][expect["slots"] >= 0]
        assert len(set(live.tolist())) == live.size


# ----------------------------------------------------------------- append
def _runs(rng, page, pool, counts, firsts):
    """Slots of runs of rows: request i writes counts[i] rows from row firsts[i] of a page of its own on."""
    order, slots, at = rng.permutation(pool), [], 0
    for n, f in zip(counts, firsts):
        slots += [int(order[at + p // page]) * page + p % page for p in range(f, f + n)]
        at += ok.pages_of(f + n, page)
    assert at <= pool
    return np.array(slots)


def _check_append(rng, slots, page, kv, dim, pool, rotary, positions=None, spread=1.0):
    tokens = len(slots)
    heads = 3 * kv  # k and v are columns of a q | k | v matrix
    qkv = (rng.standard_normal((tokens, (heads + 2 * kv) * dim)) * spread).astype(np.float32)
    positions = rng.integers(0, 500, tokens) if positions is None else positions
    rope = _rope(500, rotary) if rotary else None
    codes = rng.integers(-127, 128, (2, pool, kv, page, dim)).astype(np.int8)
    scales = (rng.uniform(0.5, 1.5, (2, pool, kv)) * 0.025 * spread).astype(np.float32)
    g = torch.from_numpy(qkv).cuda()
    cache = lq.Kv8Cache(*(torch.from_numpy(c).cuda() for c in codes), *(torch.from_numpy(s).cuda() for s in scales))
    k, v = g[:, heads * dim:(heads + kv) * dim], g[:, (heads + kv) * dim:]
    lq.kv8_append(k, v, cache, _i32(slots), _i32(positions), rope=_rope_cuda(rope))
    torch.cuda.synchronize()
    live = np.asarray(slots) >= 0
    rows = qkv[:, heads * dim:].reshape(tokens, 2, kv, dim)
    for side, x, got, got_scale in ((0, ok.rotate(rows[:, 0], positions, rope), cache.k, cache.k_scale),
                                    (1, rows[:, 1], cache.v, cache.v_scale)):
        expect, expect_scale, unrounded = ok.append(x, np.where(live, slots, -1), codes[side], scales[side])
        got, got_scale = got.cpu().numpy(), got_scale.cpu().numpy()
        assert np.all(np.abs(got_scale - expect_scale) <= 8 * U * expect_scale)
        differ = got != expect
        tie = np.abs(np.abs(unrounded - np.floor(unrounded)) - 0.5) < 127 * 16 * U
        assert not np.any(differ & ~tie), f"{int((differ & ~tie).sum())} codes differ"
        assert np.all(np.abs(got.astype(int) - expect) <= 1)
    return cache


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("rotate", ["none", "part", "all"])
def test_append_pages_and_heads(cuda_device, dim, page, rotate):
    rng = np.random.default_rng(dim * 1000 + page)
    rotary = {"none": 0, "part": dim // 4 // 8 * 8 or 8, "all": dim}[rotate]
    counts = [1, page, 2 * page + 3, page - 1, 5, 1, 1]
    firsts = [0, 0, page // 2, 1, page - 2, page - 1, 3]
    slots = _runs(rng, page, 16, counts, firsts)
    _check_append(rng, slots, page, 2, dim, 16, rotary)
    assert _status_ok()


@pytest.mark.parametrize("tokens,kv", [(1, 1), (1, 5), (700, 1), (3001, 8)])
def test_append_row_counts(cuda_device, tokens, kv):
    rng = np.random.default_rng(tokens)
    page = 64
    slots = _runs(rng, page, ok.pages_of(tokens + 7, page), [tokens], [7])
    _check_append(rng, slots, page, kv, 64, ok.pages_of(tokens + 7, page), 64)


def test_append_many_single_rows(cuda_device):
    # A decode step: every row in a page of its own, somewhere inside it.
    rng = np.random.default_rng(9)
    for tokens in (64, 700):
        slots = rng.permutation(tokens) * 32 + rng.integers(0, 32, tokens)
        _check_append(rng, slots, 32, 4, 64, tokens, 64)


def test_append_skips_rows_without_a_slot(cuda_device):
    rng = np.random.default_rng(11)
    slots = _runs(rng, 32, 8, [20, 40, 1], [4, 0, 31])
    slots = np.concatenate([[-1, -1], slots[:20], [-1], slots[20:], [-1] * 5])
    _check_append(rng, slots, 32, 2, 64, 8, 64)
    # What a skipped row holds does not matter, nor does its position.
    k = torch.full((3, 64), float("nan"), device="cuda")
    k[1] = 2.0
    cache = lq.Kv8Cache.empty(2, 1, 16, 64)
    cache.k_scale.fill_(float("nan"))  # a fresh page's old scale is not read
    rope = _rope_cuda(_rope(4, 64))
    lq.kv8_append(k, k, cache, _i32([-1, 16, -1]), _i32([-7, 0, 900]), rope=rope)
    assert torch.all(cache.v[1, 0, 0] == 127) and float(cache.v_scale[1, 0]) == np.float32(2.0) / np.float32(127)
    assert torch.all(cache.k[1, 0, 0] == 127)
    assert _status_ok()


def test_append_reports_slots_outside_the_pool(cuda_device):
    cache = lq.Kv8Cache.empty(2, 1, 16, 32)
    for t in (cache.k, cache.v):
        t.fill_(3)
    before = cache.k.clone()
    k = torch.ones((3, 32), device="cuda")
    lq.kv8_append(k, k, cache, _i32([32, -5, 2**31 - 1]))
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    assert torch.equal(cache.k, before) and torch.equal(cache.v, before)
    lq.kv8_append(k[:1], k[:1], cache, _i32([0]), _i32([9]), rope=_rope_cuda(_rope(9, 32)))  # a position past the tables
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID


def test_append_zero_and_not_a_number(cuda_device):
    cache = lq.Kv8Cache.empty(3, 1, 16, 32)
    k = torch.zeros((3, 32), device="cuda")
    k[1, 5] = float("nan")
    k[2, 7] = float("inf")
    lq.kv8_append(k, k, cache, _i32([0, 16, 32]))
    s = cache.k_scale[:, 0].tolist()
    assert s[0] == np.float32(1e-12) and torch.all(cache.k[0, 0, 0] == 0)
    assert np.isnan(s[1]) and np.isinf(s[2])  # the page shows what went in


def test_append_rounds_each_step_to_float(cuda_device):
    # code = rint(x * (1 / scale)) with every step rounded to float: bit for bit, products that round to a half included.
    rng = np.random.default_rng(12)
    tokens, kv, dim, page = 4096, 4, 64, 64
    x = rng.standard_normal((2, tokens, kv * dim)).astype(np.float32)
    cos, sin = _rope(tokens, dim)
    cache = lq.Kv8Cache.empty(tokens // page, kv, page, dim)
    k, v = (torch.from_numpy(a).cuda() for a in x)
    lq.kv8_append(k, v, cache, _i32(np.arange(tokens)), _i32(np.arange(tokens)), rope=_rope_cuda((cos, sin)))
    turned = x[0].reshape(tokens, kv, dim).copy()
    a, b = turned[..., :dim // 2].copy(), turned[..., dim // 2:].copy()
    turned[..., :dim // 2] = a * cos[:, None] - b * sin[:, None]
    turned[..., dim // 2:] = b * cos[:, None] + a * sin[:, None]
    for rows, codes, scales in ((turned, cache.k, cache.k_scale), (x[1].reshape(tokens, kv, dim), cache.v, cache.v_scale)):
        rows = rows.reshape(-1, page, kv, dim).transpose(0, 2, 1, 3)  # [pages, kv, page, dim]
        scale = np.maximum(np.abs(rows).max(axis=(2, 3)) / np.float32(127), np.float32(1e-12))
        expect = np.rint(rows * (np.float32(1) / scale)[:, :, None, None])
        assert np.array_equal(scales.cpu().numpy(), scale)
        assert np.array_equal(codes.cpu().numpy(), expect)


def test_append_twice_is_append_once(cuda_device):
    rng = np.random.default_rng(3)
    cache = _check_append(rng, _runs(rng, 16, 6, [30, 9], [5, 11]), 16, 2, 64, 6, 0)
    k = torch.randn((9, 128), device="cuda")
    slots = _i32(np.arange(20, 29))
    lq.kv8_append(k, k, cache, slots)
    once = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    lq.kv8_append(k, k, cache, slots)
    assert all(torch.equal(a, b) for a, b in zip(once, (cache.k, cache.v, cache.k_scale, cache.v_scale)))


# -------------------------------------------------------------- attention
class _Batch:
    """A step over random caches: lists of cached and new tokens per request."""

    def __init__(self, rng, context, new, page, kv, group, dim, rotary=0, lengths=None, spread=1.0, pad=0, spare=2):
        self.rng, self.page, self.kv, self.group, self.dim = rng, page, kv, group, dim
        self.context, self.new = list(context), list(new)
        self.lengths = [c + n for c, n in zip(context, new)] if lengths is None else list(lengths)
        held = [ok.pages_of(n, page) for n in self.lengths]
        self.pool = sum(held) + spare
        order = rng.permutation(self.pool)
        self.table = np.full((len(held), max(held, default=0) + 1), -1)
        at = 0
        for s, b in enumerate(held):
            self.table[s, :b] = order[at:at + b]
            at += b
        self.unused = order[at:]
        self.codes = np.clip(np.rint(rng.standard_normal((2, self.pool, kv, page, dim)) * 38), -127, 127).astype(np.int8)
        self.scales = (rng.uniform(0.5, 1.5, (2, self.pool, kv)) * 0.025).astype(np.float32)
        self.scales[:, self.unused] = np.nan  # pages nobody holds are not read
        self.tokens = sum(new) + pad
        self.q = (rng.standard_normal((self.tokens, kv * group * dim)) * spread).astype(np.float32)
        self.rope = _rope(max([c + n for c, n in zip(context, new)] + [1]), rotary) if rotary else None
        self.scale = dim ** -0.5
        self.cache = lq.Kv8Cache(*(torch.from_numpy(c).cuda() for c in self.codes),
                                 *(torch.from_numpy(s).cuda() for s in self.scales))
        prefix = lambda x: _i32(np.concatenate([[0], np.cumsum(np.asarray(x, dtype=np.int64))]))  # noqa: E731
        self.plan = lq.Kv8Plan(_i32(self.context), _i32(self.lengths), prefix(new), prefix(held), _i32(self.table),
                               self.tokens, max(new, default=0))

    def run(self, q=None, **more):
        q = torch.from_numpy(self.q).cuda() if q is None else q
        return lq.kv8_attention(q, self.cache, self.plan, self.scale, rope=_rope_cuda(self.rope), **more)

    def check(self, got=None):
        got = (self.run() if got is None else got).cpu().numpy().astype(np.float64)
        expect, bound = np.zeros_like(got), np.zeros_like(got)
        heads = self.kv * self.group
        at = 0
        for s, (c, n) in enumerate(zip(self.context, self.new)):
            positions = np.arange(c, c + n)
            q = ok.rotate(self.q[at:at + n].reshape(n, heads, self.dim), positions, self.rope)
            held = self.table[s, :ok.pages_of(self.lengths[s], self.page)]
            for h in range(self.kv):
                k, v = (self.codes[i][held, h].reshape(-1, self.dim).astype(np.float64) *
                        np.repeat(self.scales[i][held, h].astype(np.float64), self.page)[:, None] for i in range(2))
                out, reach = ok.attention(q[:, h * self.group:(h + 1) * self.group],
                                          np.minimum(positions + 1, self.lengths[s]), k, v, self.scale)
                cols = slice(h * self.group * self.dim, (h + 1) * self.group * self.dim)
                expect[at:at + n, cols] = out.reshape(n, self.group * self.dim)
                largest = np.abs(v[:self.lengths[s]]).max(initial=0.0)
                err = largest * (2 * (self.dim + 16) * reach + 64) * U
                bound[at:at + n, cols] = np.repeat(err, self.dim, axis=1)
            at += n
        got, expect, bound = got[:at], expect[:at], bound[:at]
        off = np.abs(got - expect)
        assert np.all(off <= bound), f"largest error {off.max()}, {int((off > bound).sum())} of {off.size} too far"
        assert np.linalg.norm(off) <= 1e-5 * np.linalg.norm(expect)
        assert _status_ok()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 12, 16, 40])
def test_attention_decode_heads(cuda_device, dim, group):
    rng = np.random.default_rng(dim + group)
    _Batch(rng, [0, 1, 15, 63, 64, 300], [1] * 6, 64, 2, group, dim, rotary=dim).check()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("new", [1, 2, 5, 9])
def test_attention_decode_pages(cuda_device, page, new):
    rng = np.random.default_rng(page + new)
    context = [0, 1, page - 1, page, page + 1, 3 * page - new, 1000, 17]
    _Batch(rng, context, [new] * 8, page, 3, 4, 64, rotary=32).check()
    _Batch(rng, context, [new, 0, 1, new, 0, new, 1, 0], page, 1, 8, 128).check()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("group,page", [(1, 64), (3, 16), (8, 64), (8, 128), (5, 32)])
def test_attention_prompts(cuda_device, dim, group, page):
    rng = np.random.default_rng(dim + group + page)
    _Batch(rng, [0, 0, 100, 37, 513], [130, 1, 65, 200, 33], page, 2, group, dim, rotary=dim).check()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("kv,group,page", [(32, 1, 64), (12, 3, 16), (8, 8, 64), (4, 16, 128), (13, 5, 32)])
def test_attention_prompts_of_many_heads(cuda_device, dim, kv, group, page):
    # Enough query rows for the kernel that tiles them by 128, whatever the requests' lengths.
    rng = np.random.default_rng(dim + kv + page)
    _Batch(rng, [0, 300, 95, 0, 17], [97, 1, 33, 0, 64], page, kv, group, dim, rotary=dim // 2).check()


@pytest.mark.parametrize("new", [40, 47, 48, 49, 95, 96, 97, 193])
def test_attention_tile_edges(cuda_device, new):
    rng = np.random.default_rng(new)
    _Batch(rng, [0, 96 - new % 96], [new, new], 16, 16, 4, 64, rotary=64).check()
    _Batch(rng, [64, 500], [new, 1], 128, 16, 6, 128).check()


@pytest.mark.parametrize("spread", [0.0, 1e-6, 12.0, 40.0])
def test_attention_tile_score_ranges(cuda_device, spread):
    # Later keys outweigh earlier ones by orders of magnitude, tile after tile: the running reference has to follow.
    rng = np.random.default_rng(33)
    b = _Batch(rng, [400, 0], [50, 50], 16, 8, 8, 64, spread=spread)
    rise = np.linspace(-3, 0, b.pool)[np.argsort(np.argsort(rng.random(b.pool)))]
    b.scales[0] *= 10.0 ** rise[:, None].astype(np.float32)
    b.scales[1] *= 10.0 ** (2 * rise[::-1, None]).astype(np.float32)
    b.cache.k_scale.copy_(torch.from_numpy(b.scales[0]))
    b.cache.v_scale.copy_(torch.from_numpy(b.scales[1]))
    b.check()


def test_attention_tiles_where_nothing_is_seen(cuda_device):
    rng = np.random.default_rng(34)
    b = _Batch(rng, [0, 20, 64, 0], [60] * 4, 16, 8, 8, 64, lengths=[0, 20, 124, 0], spare=20, pad=2)
    b.q[-2:] = np.nan
    out = b.run(out=torch.full(b.q.shape, 7.0, device="cuda"))
    assert torch.all(out[:60] == 0) and torch.all(out[180:240] == 0) and torch.all(out[-2:] == 7.0)
    b.check(out)
    b.plan.table[1, 1] = b.pool  # out of range: hidden and reported
    b.plan.table[2, 0] = -5
    out = b.run()
    assert torch.isfinite(out).all()
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    b.cache.k_scale[int(b.table[2, 3]), 0] = float("nan")
    out = b.run().reshape(-1, 8, 8 * 64)
    assert torch.isnan(out[120 + 48:180, 0]).all() and torch.isfinite(out[:-2, 1:]).all()
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [16, 127, 128, 129, 255, 257, 600])
def test_attention_prompt_lengths(cuda_device, dim, new):
    rng = np.random.default_rng(new)
    _Batch(rng, [0], [new], 64, 1, 2, dim, rotary=dim).check()
    _Batch(rng, [new], [new], 16, 2, 1, dim).check()


def test_attention_long_caches(cuda_device):
    rng = np.random.default_rng(21)
    _Batch(rng, [40000, 3, 9001], [1, 1, 1], 128, 2, 8, 64, rotary=64).check()
    _Batch(rng, [20000, 500], [2, 3], 16, 1, 4, 128).check()
    _Batch(rng, [12000], [40], 32, 1, 8, 64).check()


def test_attention_many_requests(cuda_device):
    rng = np.random.default_rng(22)
    n = 700
    _Batch(rng, rng.integers(0, 90, n), rng.integers(0, 3, n), 16, 2, 2, 64, rotary=64).check()


@pytest.mark.parametrize("spread", [0.0, 1e-6, 12.0, 1e4])
def test_attention_score_ranges(cuda_device, spread):
    # Flat rows, tiny queries, near one-hot rows, and scores in the tens of thousands.
    rng = np.random.default_rng(23)
    for new in (1, 70):
        b = _Batch(rng, [0, 333], [new, new], 64, 2, 8, 64, spread=spread)
        got = b.run()
        assert torch.isfinite(got).all()
        if spread <= 12:
            b.check(got)
        else:  # the weights are one-hot up to ties: each output is (nearly) some visible value, within the pages' largest
            assert float(got.abs().max()) <= 127 * float(np.nanmax(b.scales)) * (1 + 64 * U)


def test_attention_unlike_scales(cuda_device):
    # Pages whose scales differ by twelve orders of magnitude, one of them all zeros.
    rng = np.random.default_rng(24)
    for new in (1, 40):
        b = _Batch(rng, [200, 90], [new, new], 16, 2, 4, 64, spread=0.5)
        held = b.table[0, :3]
        b.scales[1, held] = [[1e-12] * 2, [40.0] * 2, [1e-6] * 2]
        b.codes[1, held[0]] = 0
        b.cache.v_scale.copy_(torch.from_numpy(b.scales[1]))
        b.cache.v.copy_(torch.from_numpy(b.codes[1]))
        b.check()


def test_attention_rows_that_see_nothing(cuda_device):
    # Refused requests keep their old length: their queries see the cached keys only, or none at all.
    rng = np.random.default_rng(25)
    for new in (1, 3, 90):
        b = _Batch(rng, [0, 20, 64, 0], [new] * 4, 16, 2, 4, 64, lengths=[0, 20, 64 + new, 0], spare=12)
        out = b.run(out=torch.full(b.q.shape, float("nan"), device="cuda"))
        assert torch.all(out[:new] == 0) and torch.all(out[3 * new:] == 0)
        b.check(out)


def test_attention_leaves_rows_past_the_last_token(cuda_device):
    rng = np.random.default_rng(26)
    for new in (1, 60):
        b = _Batch(rng, [5, 70], [new, new], 32, 2, 4, 64, pad=3)
        b.q[-3:] = np.nan
        out = b.run(out=torch.full(b.q.shape, 7.0, device="cuda"))
        assert torch.all(out[-3:] == 7.0)
        b.check(out)


def test_attention_reports_pages_outside_the_pool(cuda_device):
    rng = np.random.default_rng(27)
    for new in (1, 50):
        b = _Batch(rng, [100, 30], [new, new], 16, 1, 4, 64)
        b.plan.table[0, 2] = b.pool
        b.plan.table[1, 0] = -1
        out = b.run()
        assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
        assert torch.isfinite(out).all()
        b.rope = _rope(40, 64)  # positions past the tables
        b.run()
        assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
        assert _status_ok()


def test_attention_not_a_number_stays_in_its_request(cuda_device):
    rng = np.random.default_rng(28)
    for new in (1, 50):
        b = _Batch(rng, [100, 30], [new, new], 16, 2, 4, 64)
        b.cache.k_scale[int(b.table[0, 1]), 0] = float("nan")
        out = b.run().reshape(2, new, 2, -1)
        assert torch.isnan(out[0, :, 0]).all()
        assert torch.isfinite(out[0, :, 1]).all() and torch.isfinite(out[1]).all()


def test_attention_columns_streams_and_repeats(cuda_device):
    rng = np.random.default_rng(29)
    for context, new in (([700, 3000, 12], [1, 1, 1]), ([100, 0, 7], [90, 140, 1])):
        b = _Batch(rng, context, new, 64, 4, 8, 64, rotary=64)
        width = b.q.shape[1]
        wide = torch.randn((b.tokens, width + 512), device="cuda")
        wide[:, :width] = torch.from_numpy(b.q).cuda()
        ws = lq.Kv8Workspace()
        first = b.run(wide[:, :width], workspace=ws)
        b.check(first)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            again = [b.run(wide[:, :width], workspace=ws) for _ in range(3)]
        other.synchronize()
        assert all(torch.equal(first, x) for x in again)  # the same bits every time


@pytest.mark.parametrize("dim,group,page", [(32, 8, 64), (64, 8, 16), (96, 2, 32), (128, 3, 16), (128, 8, 128)])
def test_attention_repeats_bit_for_bit(cuda_device, dim, group, page):
    # Enough blocks and tiles for an unordered read or write to show.
    rng = np.random.default_rng(dim + group)
    for context, new in (([3000, 10, 1500, 4000], [700, 1300, 300, 900]), ([9000, 20000, 300, 7000], [1, 1, 1, 1])):
        b = _Batch(rng, context, new, page, 4, group, dim, rotary=dim)
        q = torch.from_numpy(b.q).cuda()
        first = b.run(q)
        assert torch.isfinite(first).all()
        for _ in range(12):
            assert torch.equal(first, b.run(q))
    assert _status_ok()


def test_attention_code_offsets_past_32_bits(cuda_device):
    # A pool of 2.4 GB of keys: the held pages lie at both of its ends.
    page, kv, dim = 128, 4, 128
    pages = 2_400_000_000 // (page * kv * dim) + 1
    cache = lq.Kv8Cache.empty(pages, kv, page, dim)
    rng = np.random.default_rng(30)
    for context, new in (([300], [1]), ([200], [40])):
        b = _Batch(rng, context, new, page, kv, 2, dim, spare=0)
        place = [pages - 1 - i if i % 2 else i for i in range(b.pool)]
        for big, small in ((cache.k, b.cache.k), (cache.v, b.cache.v), (cache.k_scale, b.cache.k_scale),
                           (cache.v_scale, b.cache.v_scale)):
            big[place] = small
        b.plan.table.copy_(torch.where(b.plan.table >= 0, _i32(place)[b.plan.table.clamp(min=0).long()], -1))
        b.check(lq.kv8_attention(torch.from_numpy(b.q).cuda(), cache, b.plan, b.scale))
        k = torch.randn((2, kv * dim), device="cuda")
        lq.kv8_append(k, k, cache, _i32([(pages - 3) * page, (pages - 3) * page + 1]))
        back = cache.k[pages - 3, :, :2].float() * cache.k_scale[pages - 3][:, None, None]
        assert float((back.permute(1, 0, 2).reshape(2, -1) - k).abs().max()) <= 0.51 * float(cache.k_scale[pages - 3].max())


def test_step_in_a_graph(cuda_device):
    # Plan, append and attention captured once and replayed while the requests grow.
    rng = np.random.default_rng(31)
    requests, page, kv, group, dim = 5, 16, 2, 4, 64
    table = torch.full((requests, 20), -1, dtype=torch.int32, device="cuda")
    free = _i32(rng.permutation(100))
    length, new, taken = _i32([0] * requests), _i32([1] * requests), _i32([0])
    cache = lq.Kv8Cache.empty(100, kv, page, dim)
    rope = _rope_cuda(_rope(320, dim))
    qkv = torch.zeros((requests, (kv * group + 2 * kv) * dim), device="cuda")
    q, k, v = qkv.split([kv * group * dim, kv * dim, kv * dim], dim=1)
    out, ws, plan = torch.zeros(q.shape, device="cuda"), lq.Kv8Workspace(), None

    def step():
        nonlocal plan
        for flags in (_lib.LEAFQ_FLAG_PDL,):
            plan = lq.kv8_plan(length, new, table, free, taken, page, requests, max_tokens=1, out=plan, flags=flags)
            lq.kv8_append(k, v, cache, plan.slots, plan.positions, rope=rope, flags=flags)
            lq.kv8_attention(q, cache, plan, dim ** -0.5, rope=rope, out=out, workspace=ws, flags=flags)
            length.copy_(plan.lengths)
            taken.copy_(plan.taken)

    step()
    torch.cuda.synchronize()
    length.zero_()
    taken.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    seen = []
    for t in range(40):
        row = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(t))
        qkv.copy_(row)
        seen.append(row.numpy())
        graph.replay()
    torch.cuda.synchronize()
    assert length.tolist() == [40] * requests and int(taken.item()) == 3 * requests
    rows = np.stack(seen)  # [steps, requests, width]
    rope = _rope(320, dim)
    for s in range(requests):
        x = rows[:, s].reshape(40, -1, dim)
        turned = ok.rotate(x[:, :kv * group + kv], np.arange(40), rope)
        held = table[s, :3].tolist()
        for h in range(kv):
            keys = (cache.k[held, h].float() * cache.k_scale[held, h][:, None, None]).reshape(-1, dim)[:40].cpu().numpy()
            values = (cache.v[held, h].float() * cache.v_scale[held, h][:, None, None]).reshape(-1, dim)[:40].cpu().numpy()
            # What the cache holds is what went in, to its own rounding: half a code each time a scale grew.
            assert np.abs(keys - turned[:, kv * group + h]).max() <= 8 * float(cache.k_scale[held, h].max())
            expect, _ = ok.attention(turned[-1:, h * group:(h + 1) * group], [40], keys.astype(np.float64),
                                     values.astype(np.float64), dim ** -0.5)
            got = out[s].reshape(kv, group, dim)[h].cpu().numpy()
            assert np.linalg.norm(got - expect[0]) <= 1e-5 * np.linalg.norm(expect[0])
    assert _status_ok()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("context,new", [([3000], [256]), ([0, 2500, 90, 700], [3, 150, 64, 40]), ([1200, 5000], [31, 225])])
def test_attention_few_row_tiles_over_long_caches(cuda_device, dim, context, new):
    # Fewer row tiles than blocks: each is cut along its keys and its parts are joined.
    rng = np.random.default_rng(dim + len(new))
    batch = _Batch(rng, context, new, 16, 2, 8, dim, rotary=dim)
    first = batch.run()
    batch.check(first)
    for _ in range(3):
        assert torch.equal(batch.run(), first)
    assert _status_ok()


def test_attention_parts_with_hidden_rows_and_values_that_are_no_numbers(cuda_device):
    rng = np.random.default_rng(77)
    batch = _Batch(rng, [4000, 900], [130, 126], 64, 2, 8, 64, lengths=[2100, 0])
    batch.check()
    batch.q[:] *= 40.0  # one key has nearly all the weight, in some part
    batch.check()
    q = batch.q.copy()
    q[5, 3] = np.nan
    got = batch.run(torch.from_numpy(q).cuda())
    assert torch.isnan(got[5, :64]).all() and not torch.isnan(got[6]).any() and not torch.isnan(got[5, 64:]).any()
    assert _status_ok()


def test_attention_shapes_share_a_workspace(cuda_device):
    # Decode, draft, prompt and few-head shapes in turn: none may find another's leavings.
    rng = np.random.default_rng(78)
    batches = [_Batch(rng, [9000], [1], 64, 1, 8, 64), _Batch(rng, [3000], [200], 64, 1, 8, 64),
               _Batch(rng, [5000, 20], [1, 1], 32, 4, 2, 128), _Batch(rng, [3000], [256], 64, 2, 8, 128),
               _Batch(rng, [2000, 700], [40, 290], 16, 1, 8, 32), _Batch(rng, [6000], [4], 16, 3, 1, 96)]
    alone = [b.run() for b in batches]
    for b, y in zip(batches, alone):
        b.check(y)
    workspace = lq.Kv8Workspace("cuda")
    for order in ((0, 1, 2, 3, 4, 5), (5, 3, 1, 4, 0, 2), (1, 1, 0, 4, 4, 3)):
        for i in order:
            assert torch.equal(batches[i].run(workspace=workspace), alone[i])
    assert _status_ok()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("requests,new,page", [(70, 1, 16), (160, 2, 64), (400, 1, 32)])
def test_attention_more_heads_than_blocks(cuda_device, dim, requests, new, page):
    # Short caches, empty ones and a long one; requests that bring nothing among them.
    rng = np.random.default_rng(dim + requests)
    context = rng.integers(0, 60, requests)
    context[rng.random(requests) < 0.1] = 0
    context[requests // 3] = 4000
    fresh = np.where(rng.random(requests) < 0.1, 0, rng.integers(1, new + 1, requests))
    batch = _Batch(rng, [int(c) for c in context], [int(n) for n in fresh], page, 8, 5, dim, rotary=dim // 2)
    first = batch.run()
    batch.check(first)
    assert torch.equal(batch.run(), first)
    assert _status_ok()



def _no_counter_left(workspace):
    torch.cuda.synchronize()
    return not bool(workspace.buffer[:16384].any())  # the counters, in front of the partial results


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("requests,live,kv,group,new", [
    (256, {97: 1000}, 8, 2, 1), (112, {0: 1000}, 8, 1, 1), (320, {3: 1500, 150: 1500, 319: 1500}, 4, 8, 1),
    (24, {11: 1000}, 8, 8, 8), (200, {7: 700, 8: 40, 199: 2000}, 12, 3, 2)])
def test_attention_few_live_requests_among_idle_ones(cuda_device, dim, requests, live, kv, group, new):
    # More heads than blocks, but fewer pages of heads: no block that has none may be waited for.
    rng = np.random.default_rng(dim + requests)
    idle = _Batch(rng, [live.get(s, 0) for s in range(requests)], [new if s in live else 0 for s in range(requests)], 64, kv,
                  group, dim, rotary=dim)
    other = _Batch(rng, [3000, 50], [1, 1], 64, 2, 8, dim)
    workspace = lq.Kv8Workspace()
    for b in (idle, idle, other, idle):
        b.check(b.run(out=torch.full(b.q.shape, float("nan"), device="cuda"), workspace=workspace))
        assert _no_counter_left(workspace)


def _with_scores_near(b, level):
    """Keys whose scores are all about -level: large codes of one sign, queries of the other."""
    b.codes[0] = b.rng.integers(64, 128, b.codes[0].shape)
    b.q = -np.abs(b.q)
    b.scales[0] = np.where(np.isnan(b.scales[0]), np.nan, level / (b.scale * 0.8 * 95.5 * b.dim))
    b.cache.k.copy_(torch.from_numpy(b.codes[0]))
    b.cache.k_scale.copy_(torch.from_numpy(b.scales[0]))
    return b


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("context,new,group", [([27, 5], [9, 3], 1), ([61, 2045], [6, 7], 1), ([30, 4090, 94], [4, 9, 2], 3)])
def test_attention_low_scores_beside_chunks_that_a_row_does_not_see(cuda_device, dim, context, new, group):
    # Keys that only the later rows of a block see are no reference for the earlier ones.
    rng = np.random.default_rng(dim + group)
    for heads in (1, 2):
        _with_scores_near(_Batch(rng, context, new, 16, heads, group, dim), 140.0).check()


@pytest.mark.parametrize("new,kv,group", [(1, 2, 4), (60, 8, 8)])
def test_attention_low_scores_behind_hidden_pages(cuda_device, new, kv, group):
    # Pages outside the pool hide their keys: what is seen behind them is weighed as if they were not there.
    rng = np.random.default_rng(35)
    b = _with_scores_near(_Batch(rng, [300], [new], 16, kv, group, 64), 140.0)
    b.plan.table[0, :8] = -1
    got = b.run().reshape(new, kv, group, 64).cpu().numpy()
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    held = b.table[0, 8:ok.pages_of(300 + new, 16)]
    for h in range(kv):
        k, v = (b.codes[i][held, h].reshape(-1, 64) * np.repeat(b.scales[i][held, h].astype(np.float64), 16)[:, None]
                for i in range(2))
        q = b.q.reshape(new, kv, group, 64)[:, h].astype(np.float64)
        expect, reach = ok.attention(q, np.arange(300, 300 + new) + 1 - 128, k, v, b.scale)
        assert np.all(np.abs(got[:, h] - expect) <= np.abs(v).max() * (2 * (64 + 16) * reach[..., None] + 64) * U)


@pytest.mark.parametrize("requests,kv,dim", [(74, 4, 64), (37, 8, 64), (111, 4, 128), (37, 12, 96), (296, 1, 32)])
def test_attention_as_many_heads_as_blocks(cuda_device, requests, kv, dim):
    # One piece a head is all that the blocks can take, whatever the longest heads' length.
    page, most = 16, 700
    cache = lq.Kv8Cache.empty(most, kv, page, dim)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.copy_(torch.randint(-127, 128, codes.shape, device="cuda", dtype=torch.int8))
        scale.fill_(0.02)
    table = torch.arange(most, dtype=torch.int32, device="cuda").repeat(requests, 1)
    q = torch.randn((requests, kv * dim), device="cuda")
    workspace = lq.Kv8Workspace()
    offsets = _i32(np.arange(requests + 1))
    alone = {}
    for held in list(range(26, 400)) + [511, 513, 699, 700]:
        pages = np.where(np.arange(requests) % 2 == 0, held, 1 + np.arange(requests) % 5)
        lengths = pages * page
        plan = lq.Kv8Plan(_i32(lengths - 1), _i32(lengths), offsets, _i32(np.concatenate([[0], np.cumsum(pages)])), table,
                          requests, 1)
        out = torch.full(q.shape, float("nan"), device="cuda")
        lq.kv8_attention(q, cache, plan, dim ** -0.5, out=out, workspace=workspace)
        assert torch.isfinite(out).all(), f"{held} pages"
        assert _no_counter_left(workspace), f"{held} pages"
        alone.setdefault("short", out[1::2])
        assert torch.equal(alone["short"], out[1::2])
    assert _status_ok()


def test_plan_that_is_reused_takes_the_new_bound(cuda_device):
    # The rows stay the same, one request's share of them does not: 64 requests of one token, then one of 60.
    rng = np.random.default_rng(36)
    requests, page, kv, group, dim = 64, 16, 2, 4, 64
    context, table = _i32([0] * requests), torch.full((requests, 8), -1, dtype=torch.int32, device="cuda")
    free, taken = _i32(rng.permutation(requests * 8)), _i32([0])
    cache = lq.Kv8Cache.empty(requests * 8, kv, page, dim)
    rows = torch.randn((requests, kv * dim), device="cuda")
    q = torch.randn((requests, kv * group * dim), device="cuda")
    plan = lq.kv8_plan(context, _i32([1] * requests), table, free, taken, page, requests, max_tokens=1)
    lq.kv8_append(rows, rows, cache, plan.slots)
    lq.kv8_attention(q, cache, plan, dim ** -0.5)
    context.copy_(plan.lengths)
    taken.copy_(plan.taken)
    new = [0] * requests
    new[5] = 60
    again = lq.kv8_plan(context, _i32(new), table, free, taken, page, requests, max_tokens=60, out=plan)
    assert again is plan and plan.max_tokens == 60
    lq.kv8_append(rows, rows, cache, plan.slots)
    out = lq.kv8_attention(q, cache, plan, dim ** -0.5, out=torch.full(q.shape, float("nan"), device="cuda"))
    fresh = lq.kv8_plan(context, _i32(new), table.clone(), free, taken, page, requests, max_tokens=60)
    expect = lq.kv8_attention(q, cache, fresh, dim ** -0.5)
    assert torch.isfinite(out[:60]).all() and torch.equal(out[:60], expect[:60])
    held = table[5, :4].long()
    k, v = ((c[held].float() * s[held][:, :, None, None]).permute(1, 0, 2, 3).reshape(kv, -1, dim).double().cpu().numpy()
            for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    for h in range(kv):
        x = q[:60].reshape(60, kv, group, dim)[:, h].double().cpu().numpy()
        exact, reach = ok.attention(x, np.arange(60) + 2, k[h], v[h], dim ** -0.5)
        got = out[:60].reshape(60, kv, group, dim)[:, h].cpu().numpy()
        assert np.all(np.abs(got - exact) <= np.abs(v[h]).max() * (2 * (dim + 16) * reach[..., None] + 64) * U)
    # Without a bound it is the step's rows again.
    assert lq.kv8_plan(context, _i32(new), table, free, taken, page, requests, out=plan).max_tokens == requests
    assert plan.desc.max_tokens == requests
    with pytest.raises(lq.LeafError, match="negative"):
        lq.kv8_plan(context, _i32(new), table, free, taken, page, requests, max_tokens=-1, out=plan)
    assert _status_ok()


def test_graph_replays_after_its_workspace_has_grown(cuda_device):
    rng = np.random.default_rng(38)
    decode, prompt = _Batch(rng, [9000, 300], [1, 1], 64, 2, 8, 64), _Batch(rng, [40], [700], 64, 4, 8, 64)
    workspace = lq.Kv8Workspace()
    q, out = torch.from_numpy(decode.q).cuda(), torch.zeros(decode.q.shape, device="cuda")
    decode.run(q, out=out, workspace=workspace)
    expect = out.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode.run(q, out=out, workspace=workspace)
    first = workspace.buffer.data_ptr()
    size = workspace.buffer.numel()
    prompt.check(prompt.run(workspace=workspace))
    assert workspace.buffer.data_ptr() != first
    others = [torch.full((size,), 77, dtype=torch.uint8, device="cuda") for _ in range(4)]
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(out, expect)
    assert all(bool((t == 77).all()) for t in others)
    prompt.check(prompt.run(workspace=workspace))
    assert _no_counter_left(workspace)


@pytest.mark.parametrize("new,kv,group,dim", [(1, 2, 4, 64), (3, 4, 2, 128), (40, 8, 8, 64), (60, 8, 6, 128), (260, 1, 8, 96)])
@pytest.mark.parametrize("kind", ["first", "all", "last", "small", "beside large", "steps"])
def test_attention_value_scales_of_zero_and_small_ones(cuda_device, new, kv, group, dim, kind):
    # A page whose values are all zero counts in the sum of the weights as any other.
    rng = np.random.default_rng(new + dim)
    b = _Batch(rng, [1500, 200], [new, new], 16, kv, group, dim, spread=0.5)
    for held in ([int(p) for p in row if p >= 0] for row in b.table):
        pages = np.arange(len(held))
        if kind == "first":
            b.scales[1, held[:5]] = 0.0
        elif kind == "all":
            b.scales[1, held] = 0.0
        elif kind == "last":
            b.scales[1, held[-3:]] = 0.0
        elif kind == "small":
            b.scales[1, held] *= 2.0 ** -80
        elif kind == "beside large":
            b.scales[1, held] *= np.where(pages % 3 == 0, 0.0, 1e14)[:, None].astype(np.float32)
        else:
            b.scales[1, held] = (10.0 ** (-7.0 * (4 - pages % 5)))[:, None]
    b.cache.v_scale.copy_(torch.from_numpy(b.scales[1]))
    b.check()


@pytest.mark.parametrize("new,kv,group", [(1, 2, 4), (70, 8, 8)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_values_that_are_all_no_numbers(cuda_device, new, kv, group, value):
    rng = np.random.default_rng(37)
    b = _Batch(rng, [20, 6], [new, new], 16, kv, group, 64)
    b.cache.v_scale[[int(p) for p in b.table[0] if p >= 0], 1] = value
    got = b.run().reshape(2, new, kv, -1)
    assert not torch.isfinite(got[0, :, 1]).any()
    assert torch.isfinite(got[0, :, 0]).all() and torch.isfinite(got[1]).all()
    assert _status_ok()


@pytest.mark.parametrize("new,kv,group,dim", [(9, 2, 1, 64), (9, 2, 1, 96), (6, 3, 4, 128), (70, 8, 8, 64), (70, 8, 6, 128), (70, 8, 8, 32)])
@pytest.mark.parametrize("which,value", [("k", float("nan")), ("v", float("nan")), ("k", float("inf")), ("v", float("inf"))])
def test_attention_rows_are_clear_of_pages_that_they_do_not_see(cuda_device, new, kv, group, dim, which, value):
    # A page of scale NaN or infinity shows in the rows that see it, not in those before it.
    rng = np.random.default_rng(new + dim)
    b = _Batch(rng, [43, 11], [new, new], 16, kv, group, dim)
    clean = b.run()
    first = 3  # request 0's page of positions 48 .., which its first five rows do not see
    scales = b.cache.k_scale if which == "k" else b.cache.v_scale
    scales[int(b.table[0, first]), 0] = value
    got = b.run()
    rows = torch.arange(b.tokens, device="cuda")
    columns = torch.arange(b.q.shape[1], device="cuda")
    sees = ((rows >= 16 * first - 43) & (rows < new))[:, None] & (columns < group * dim)
    assert torch.isfinite(got[~sees]).all()
    if not (which == "k" and value == float("inf")):  # (a score of minus infinity weighs nothing)
        assert not torch.isfinite(got[sees]).any()
    b.check(torch.where(sees, clean, got))


def test_attention_leaves_its_counters_zero_whatever_it_finds(cuda_device):
    # A call that gave up a wait leaves parts that never arrived: the next one's result is its own again.
    rng = np.random.default_rng(39)
    b = _Batch(rng, [3000], [256], 64, 2, 8, 64, rotary=64)  # 17 row tiles of 2 heads, cut along their keys
    workspace = lq.Kv8Workspace()
    b.check(b.run(workspace=workspace))
    assert _no_counter_left(workspace)
    arrivals = workspace.buffer.view(torch.int32)[2560 + 4:][:4 * 17 * 2]
    for words in (arrivals[:8], arrivals):  # of heads past the last row; of all
        words.fill_(1)
        b.run(workspace=workspace)
        assert _no_counter_left(workspace)
        b.check(b.run(workspace=workspace))


@pytest.mark.parametrize("context,new", [([700, 12, 3000], [1, 1, 1]), ([100, 0, 2000], [90, 140, 300])])
def test_step_without_early_launch_gives_the_same_bits(cuda_device, context, new):
    # Plan, append and attention with and without LEAFQ_FLAG_PDL, over the same cache.
    rng = np.random.default_rng(40)
    results = []
    for flags in (_lib.LEAFQ_FLAG_PDL, 0):
        rng = np.random.default_rng(40)
        b = _Batch(rng, context, new, 16, 4, 8, 64, rotary=64)
        free = _i32(np.concatenate([b.unused, np.arange(b.pool, b.pool + 4)]))
        table = _i32(np.where(np.arange(b.table.shape[1]) < np.array([[ok.pages_of(c, 16)] for c in context]), b.table, -1))
        # Pages of the new tokens: what the batch holds for them, in request order.
        fresh = np.concatenate([b.table[s, ok.pages_of(c, 16):ok.pages_of(c + n, 16)] for s, (c, n) in enumerate(zip(context, new))])
        plan = lq.kv8_plan(_i32(context), _i32(new), table, torch.cat((_i32(fresh), free)), _i32([0]), 16, b.tokens,
                           max_tokens=max(new), flags=flags)
        rows = [torch.from_numpy(rng.standard_normal((b.tokens, 4 * 64)).astype(np.float32)).cuda() for _ in range(2)]
        rope = _rope_cuda(b.rope)
        lq.kv8_append(*rows, b.cache, plan.slots, plan.positions, rope=rope, flags=flags)
        out = lq.kv8_attention(torch.from_numpy(b.q).cuda(), b.cache, plan, b.scale, rope=rope, flags=flags)
        held = _i32(np.unique(b.table[b.table >= 0])).long()
        results.append([plan.slots, plan.lengths, b.cache.k[held], b.cache.v_scale[held], out])
        assert torch.equal(table, _i32(b.table)) and torch.isfinite(out).all()
    assert all(torch.equal(x, y) for x, y in zip(*results))
    assert _status_ok()
