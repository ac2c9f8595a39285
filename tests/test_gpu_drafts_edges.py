"""More of the operators that check drafted tokens, on the GPU: what the sizes of test_gpu_drafts.py do not
reach, against the same 64-bit definitions (oracle/kv8.py, oracle/drafts.py).

Tolerances, with u = 2^-24:
* tree attention: as there.  Of a row that does not see a page, whatever the page's scales: 1e-5 of the largest
  value, twice what its two runs are each within of the exact one.
* compaction: equal.  A code times a scale has 32 bits at most, so the largest is exact in 64; need, the scale's
  rounding to 32 bits, the quotients and the products are then the same single operations of IEEE numbers on
  both sides.
* verification: whole numbers, equal; no request is left out.  That asks for inputs without comparisons nearer
  than the operator's error, which the seeds here give (checked from the oracle's margins in each test).  Of a
  child, p is within 2^-17 for vocabularies up to 2^17, added up from: 3.25 u of the exponent (a subtraction,
  a division, a multiplication, log2 e), whose mean under p is at most ln 2^17, 39 u; ex2's 4 u; a rescaling by
  ex2 and its rounding, 5 u each, at most 6 (four loads of 16 values a thread, two joins); 4 + 4 + 5 + 6
  additions: 92 u, 2^-17.5.  For 2^20 tokens: 45 + 4 + 34 x 5 + 48 = 267 u, 2^-15.9.  Of a draw, 2^-40 of the sum.
"""
import numpy as np
import pytest
import torch

import leaf_b200 as lq
from oracle import drafts as od
from oracle import kv8 as ok
from test_gpu_drafts import _f32, _path_of, _plan, _random_tree, _Trees, _verify_case
from test_gpu_kv8 import U, _Batch, _i32, _rope, _rope_cuda, _status_ok

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -149  # of the 32-bit numbers above zero


# ------------------------------------------------------------ verification
def _judged(trees, logits, ids, accept, sample, heat, q, child=2.0 ** -17):
    """The oracle's verdicts, of inputs that no comparison's error can turn."""
    verdicts, at = [], 0
    for s, parents in enumerate(trees):
        rows = slice(at, at + len(parents))
        path, tokens, near = od.verify(logits[rows], ids[rows], parents, accept[rows], sample[s], heat[s], None if q is None else q[rows])
        assert near[0] >= child and near[1] >= 2.0 ** -40, f"request {s} is nearer than the operator's error: {near}"
        verdicts.append((path, tokens))
        at += len(parents)
    return verdicts


def _same_verdicts(got, verdicts):
    path, tokens, kept, nxt = (t.cpu().numpy() for t in (got.path, got.tokens, got.kept, got.next))
    for s, (way, drawn) in enumerate(verdicts):
        assert kept[s] == len(way) and path[s].tolist() == way + [-1] * (path.shape[1] - len(way)), s
        assert tokens[s].tolist() == drawn + [-1] * (path.shape[1] - len(way)) and nxt[s] == (drawn[-1] if drawn else -1), s
    assert _status_ok()


def _rows_cuda(x, stride=0):
    """On the GPU, rows `stride` floats apart where it is given."""
    if not stride:
        return _f32(x)
    wide = torch.full((x.shape[0], stride), float("nan"), device="cuda")
    wide[:, :x.shape[1]] = torch.from_numpy(x).cuda()
    return wide[:, :x.shape[1]]


def _inputs(case, stride=0):
    logits, ids, accept, sample, heat, q = case
    return [_rows_cuda(logits, stride), _i32(ids), _f32(accept), _f32(sample), _f32(heat), None if q is None else _rows_cuda(q, stride)]


def _call(trees, tensors, plan=None, parents=None, out=None):
    plan = _plan([0] * len(trees), trees) if plan is None else plan
    parents = _i32([p for t in trees for p in t]) if parents is None else parents
    logits, ids, accept, sample, heat, q = tensors
    return lq.verify_drafts(logits, ids, parents, plan, accept, sample, heat, draft_probs=q, out=out)


def _batch_trees(rng, requests, large):
    trees = [_random_tree(rng, int(n), "near") if n else [] for n in rng.integers(0, 8, requests)]
    trees[0] = _random_tree(rng, 6, "binary")
    if large:  # more rows than are summed up ahead
        trees[-1] = _random_tree(rng, 30, "near")
    return trees


# Clusters of two, four and eight blocks a request (from 6,145, 12,289 and 24,577 tokens on), on both sides of as many
# blocks as there are SMs, where the rows' sums are taken ahead; and a batch of several waves.
BATCHES = [(6145, 74), (6145, 75), (12289, 37), (12289, 38), (24577, 18), (24577, 19), (24577, 130), (100003, 20)]


def _batch_case(vocab, requests, probs, large):
    rng = np.random.default_rng(vocab + requests + 2 * probs + large)
    trees = _batch_trees(rng, requests, large)
    return trees, _verify_case(rng, trees, vocab, probs, greedy=0.2)


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab,requests", BATCHES)
def test_verify_batches_of_several_blocks_a_request(cuda_device, vocab, requests, probs, large):
    trees, case = _batch_case(vocab, requests, probs, large)
    verdicts = _judged(trees, *case)
    _same_verdicts(_call(trees, _inputs(case)), verdicts)
    _same_verdicts(_call(trees, _inputs(case, stride=vocab + 3)), verdicts)  # no two rows aligned alike


def _star_case(vocab, probs, n):
    # Drafts that the target hardly ever takes, some of them several times: a rejection for nearly every child.
    rng = np.random.default_rng(vocab + n + probs)
    requests = 6
    trees = [[-1] + [0] * (n - 1)] * requests
    logits, _, accept, sample, heat, _ = _verify_case(rng, trees, vocab, False)
    ids = rng.integers(0, vocab, requests * n)
    ids[rng.random(ids.size) < 0.3] = ids[5]
    accept = rng.uniform(0.7, 1.0, accept.shape).astype(np.float32)
    q = np.full((requests * n, vocab), 1 / vocab, np.float32) if probs else None
    return trees, (logits, ids, accept, sample, heat, q)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab,n", [(6145, 60), (12289, 60), (24577, 7), (24577, 60)])
def test_verify_many_rejections_over_several_blocks(cuda_device, vocab, n, probs):
    trees, case = _star_case(vocab, probs, n)
    _same_verdicts(_call(trees, _inputs(case)), _judged(trees, *case))


def _large_case(probs):
    rng = np.random.default_rng(20 + probs)
    trees = [[-1, 0, 1, 2, 3], [-1] + [0] * 7, [-1], _random_tree(rng, 12, "near")]
    return trees, _verify_case(rng, trees, 1 << 20, probs)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_the_largest_vocabulary(cuda_device, probs):
    trees, case = _large_case(probs)
    verdicts = _judged(trees, *case, child=2.0 ** -15.5)
    _same_verdicts(_call(trees, _inputs(case)), verdicts)
    _same_verdicts(_call(trees, _inputs(case, stride=(1 << 20) + 1)), verdicts)


@pytest.mark.parametrize("vocab,blocks", [(8192, 2), (16384, 4), (32768, 8)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_verify_draws_at_the_borders_of_parts(cuda_device, vocab, blocks, shift):
    # Equal logits: token j for sample in [j / vocab, (j + 1) / vocab); the warps' parts begin at every 1 / (8 blocks).
    each = vocab // (8 * blocks)
    borders = sorted({max(0, min(vocab - 1, b * each + d)) for b in range(8 * blocks + 1) for d in (-5, -1, 0, 1, 4)})
    at = np.array(borders)
    sample = np.concatenate([at / vocab, np.nextafter(np.float32((at + 1) / vocab), np.float32(0)), [1 - 2.0 ** -24, 0.0]]).astype(np.float32)
    requests = sample.size
    logits = torch.zeros((requests, vocab + shift), device="cuda")[:, :vocab]
    got = lq.verify_drafts(logits, _i32([0] * requests), _i32([-1] * requests), _plan([0] * requests, [[-1]] * requests),
                           _f32(np.zeros(requests)), _f32(sample), _f32(np.ones(requests)))
    assert got.next.tolist() == [*borders, *borders, vocab - 1, 0] and got.kept.tolist() == [1] * requests
    # Two tokens with all the weight, in parts far apart; then the last one alone.
    rows = torch.full((5, vocab + shift), float("-inf"), device="cuda")[:, :vocab]
    rows[:4, [7, vocab - 9]] = 2.0
    rows[4, vocab - 1] = -3.0
    got = lq.verify_drafts(rows, _i32([0] * 5), _i32([-1] * 5), _plan([0] * 5, [[-1]] * 5), _f32(np.zeros(5)),
                           _f32([0.0, 0.4999, 0.5, 0.9999, 0.0]), _f32(np.ones(5)))
    assert got.next.tolist() == [7, 7, vocab - 9, vocab - 9, vocab - 1]
    assert _status_ok()


def _graph_case(seed, requests):
    rng = np.random.default_rng(seed)
    return _batch_trees(np.random.default_rng(requests), requests, False), rng


def _graph_cases(requests):
    trees, rng = _graph_case(41, requests)
    return trees, [_verify_case(rng, trees, 24577, True, greedy=0.1) for _ in range(2)]


@pytest.mark.parametrize("requests", [10, 40])
def test_verify_of_several_blocks_in_graphs_and_on_streams(cuda_device, requests):
    trees, cases = _graph_cases(requests)
    verdicts = [_judged(trees, *c) for c in cases]
    tensors = [_inputs(c) for c in cases]
    plan, parents = _plan([0] * requests, trees), _i32([p for t in trees for p in t])
    static, out = [t.clone() for t in tensors[0]], lq.Verdict(requests, plan.max_tokens, "cuda")
    _call(trees, static, plan, parents, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _call(trees, static, plan, parents, out)
    for _ in range(3):
        for values, expect in zip(tensors, verdicts):
            for a, b in zip(static, values):
                a.copy_(b)
            graph.replay()
            _same_verdicts(out, expect)
    streams, got = [torch.cuda.Stream() for _ in range(4)], [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i % 2].append(_call(trees, tensors[i % 2], plan, parents))
    torch.cuda.synchronize()
    for outs, expect in zip(got, verdicts):
        for o in outs:
            _same_verdicts(o, expect)


def _far_case():
    rng = np.random.default_rng(71)
    trees = [[-1] + [0] * 1023, [t - 1 for t in range(1024)], _random_tree(rng, 9, "near")]
    return trees, _verify_case(rng, trees[2:], 1 << 20, True)


def test_verify_rows_behind_two_thousand_million_values(cuda_device):
    # The last request's rows begin at value 2^31 of the logits and of the probabilities.
    trees, (logits, ids, accept, sample, heat, q) = _far_case()
    (path, tokens), = _judged(trees[2:], logits, ids, accept, sample, heat, q, child=2.0 ** -15.5)
    vocab = 1 << 20
    far, far_q = (torch.zeros((2048 + 9, vocab), device="cuda") for _ in range(2))
    far[2048:], far_q[2048:] = _f32(logits), _f32(q)
    far[0, 5], far[1024, 6] = 1.0, 2.0  # greedy: their drafts are token 0
    got = _call(trees, [far, _i32([0] * 2048 + ids.tolist()), _f32(np.concatenate([np.zeros(2048), accept])),
                        _f32([0.0, 0.0, sample[0]]), _f32([0.0, 0.0, heat[0]]), far_q])
    _same_verdicts(got, [([0], [5]), ([0], [6]), (path, tokens)])


# --------------------------------------------------------------- attention
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("new,kv,group", [(24, 2, 4), (60, 8, 8)])
@pytest.mark.parametrize("where", ["behind", "before"])
def test_tree_attention_rows_keep_clear_of_pages_that_they_do_not_see(cuda_device, dim, new, kv, group, where):
    # Few rows and many.  A page of drafts that some rows see and others do not: the last one, or (of trees that begin
    # without any cached token) the first, with the rows behind it in trees of their own.
    rng = np.random.default_rng(dim + new)
    context = 16 if where == "behind" else 0
    b = _Trees(rng, [context], [new], 16, kv, group, dim, kind="star", spare=8)
    if where == "behind":
        page = (context + new - 1) // 16
        hidden = range(page * 16 - context, new)
    else:
        page, hidden = 0, range(16)
        b.trees = [[-1] + [0] * 15 + [-1] + [16] * (new - 17)]
        b.parents = _i32(b.trees[0])
        b.tree = lq.kv8_tree(b.parents, b.plan)
    above = ok.tree(b.trees[0], context)[1]
    clear = [t for t, rows in enumerate(above) if not rows & set(hidden)]
    seeing = [t for t in range(new) if t not in clear]
    assert clear and seeing
    quiet = b.run()
    b.check(quiet)
    own = b.scales[:, b.table[0, page]].copy()
    scale = quiet[clear].abs().amax()
    for k_scale, v_scale in ((np.nan, own[1]), (own[0], np.nan), (np.nan, np.nan), (2000.0, own[1]), (np.inf, own[1]), (own[0], np.inf),
                             (0.0, 0.0), (own[0], 0.0)):
        b.cache.k_scale[b.table[0, page]] = torch.as_tensor(np.broadcast_to(k_scale, own[0].shape).copy(), dtype=torch.float32, device="cuda")
        b.cache.v_scale[b.table[0, page]] = torch.as_tensor(np.broadcast_to(v_scale, own[1].shape).copy(), dtype=torch.float32, device="cuda")
        out = b.run()
        assert torch.all((out[clear] - quiet[clear]).abs() <= 1e-5 * scale), (k_scale, v_scale)
        if np.isnan(k_scale).any() or np.isnan(v_scale).any():
            assert torch.isnan(out[seeing]).all()
    assert _status_ok()


def _check_visible(b, visible, positions, got):
    """Of one request: got against the definition, with the keys that each row sees."""
    got = got.cpu().numpy().astype(np.float64)
    heads, n = b.kv * b.group, b.new[0]
    q = ok.rotate(b.q.reshape(n, heads, b.dim), np.maximum(positions, 0), b.rope)
    held = b.table[0, :ok.pages_of(b.lengths[0], b.page)]
    for h in range(b.kv):
        k, v = (b.codes[i][held, h].reshape(-1, b.dim).astype(np.float64) *
                np.repeat(b.scales[i][held, h].astype(np.float64), b.page)[:, None] for i in range(2))
        out, reach = ok.tree_attention(q[:, h * b.group:(h + 1) * b.group], visible, k, v, b.scale)
        cols = slice(h * b.group * b.dim, (h + 1) * b.group * b.dim)
        bound = np.repeat(np.abs(v).max() * (2 * (b.dim + 16) * reach + 64) * U, b.dim, axis=1)
        assert np.all(np.abs(got[:, cols] - out.reshape(n, -1)) <= bound)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("context,new,kv,group", [(37, 40, 2, 4), (0, 33, 1, 3), (37, 100, 8, 8), (3000, 65, 8, 8), (0, 200, 4, 16)])
def test_tree_attention_of_any_masks(cuda_device, dim, page, context, new, kv, group):
    # Masks that no tree has: rows without themselves, bits of later rows (which count as unset) and of words behind the
    # tree's, nothing at all; positions in any order.
    rng = np.random.default_rng(context + new + dim)
    b = _Batch(rng, [context], [new], page, kv, group, dim, rotary=dim)
    bits = rng.random((new, 1024)) < rng.uniform(0, 1, (new, 1))
    bits[rng.random(new) < 0.2] = False
    masks = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    positions = rng.integers(0, context + new, new)
    positions[rng.random(new) < 0.1] = -1
    tree = lq.Kv8Tree(_i32(positions), torch.from_numpy(masks.copy()).cuda())
    out = lq.kv8_tree_attention(torch.from_numpy(b.q).cuda(), b.cache, b.plan, tree, b.scale, rope=_rope_cuda(b.rope))
    visible = np.zeros((new, ok.pages_of(context + new, page) * page), dtype=bool)
    for t in range(new):
        if positions[t] >= 0:
            visible[t, :context] = True
            visible[t, context:context + t + 1] = bits[t, :t + 1]
    assert context > 0 or (~visible.any(axis=1)).any()
    assert torch.all(out[~visible.any(axis=1)] == 0)
    _check_visible(b, visible, positions, out)
    assert _status_ok()


@pytest.mark.parametrize("new,kv,group", [(6, 2, 4), (40, 8, 8)])
def test_tree_attention_with_wide_tables(cuda_device, new, kv, group):
    # Room for far more than the requests hold, as a serving loop's tables have; what is in it is not looked at.
    rng = np.random.default_rng(new)
    b = _Trees(rng, [100, 0, 33], [new] * 3, 16, kv, group, 64, rotary=64)
    wide = torch.full((3, 5000), 2**31 - 1, dtype=torch.int32, device="cuda")
    wide[:, :b.plan.table.shape[1]] = b.plan.table
    b.plan = lq.Kv8Plan(b.plan.context, b.plan.lengths, b.plan.token_offsets, b.plan.page_offsets, wide, b.tokens, new)
    b.check()


@pytest.mark.parametrize("new,kv,group", [(6, 2, 4), (40, 8, 8), (64, 8, 4)])
def test_tree_attention_into_its_queries(cuda_device, new, kv, group):
    rng = np.random.default_rng(new)
    b = _Trees(rng, [3000, 0, 500], [new] * 3, 32, kv, group, 64, rotary=64)
    expect = b.run()
    for _ in range(3):
        q = torch.from_numpy(b.q).cuda()
        assert b.run(q, out=q) is q and torch.equal(q, expect)


@pytest.mark.parametrize("new,group", [(4, 4), (60, 8)])
def test_operators_in_pools_of_more_than_four_thousand_million_codes(cuda_device, new, group):
    # The pages of a small pool at the end of a large one: the same results.
    rng = np.random.default_rng(new)
    kv, page, dim, pool = 8, 128, 128, 33500  # 131,072 codes a page: pages from 32,768 on begin behind 2^32
    b = _Trees(rng, [500, 40], [new, new], page, kv, group, dim, rotary=dim)
    expect = b.run()
    first = pool - b.pool
    large = lq.Kv8Cache.empty(pool, kv, page, dim)
    for to, of in ((large.k, b.cache.k), (large.v, b.cache.v), (large.k_scale, b.cache.k_scale), (large.v_scale, b.cache.v_scale)):
        to[first:] = of
    table = torch.where(b.plan.table >= 0, b.plan.table + first, b.plan.table)
    plan = lq.Kv8Plan(b.plan.context, b.plan.lengths, b.plan.token_offsets, b.plan.page_offsets, table, b.tokens, new)
    q = torch.from_numpy(b.q).cuda()
    assert torch.equal(lq.kv8_tree_attention(q, large, plan, b.tree, b.scale, rope=_rope_cuda(b.rope)), expect)
    path, kept = _i32([sorted(rng.choice(new, new // 2, replace=False).tolist()) for _ in range(2)]), _i32([new // 2] * 2)
    lq.kv8_compact(lq.Kv8Layers([b.cache]), b.plan, path, kept)
    lq.kv8_compact(lq.Kv8Layers([large]), plan, path, kept)
    for got, of in ((large.k, b.cache.k), (large.v, b.cache.v)):
        assert torch.equal(got[first:], of)
    held = [p for s in range(2) for p in b.table[s, :ok.pages_of(b.lengths[s], page)].tolist()]
    for got, of in ((large.k_scale, b.cache.k_scale), (large.v_scale, b.cache.v_scale)):
        assert torch.equal(got[first:][held], of[held])
    assert _status_ok()


# ----------------------------------------------------------------- compact
def _two_pages(codes, scales, kept, path, context=14):
    cache = lq.Kv8Cache(*(torch.from_numpy(codes.copy()).cuda() for _ in range(2)), *(torch.from_numpy(scales.copy()).cuda() for _ in range(2)))
    lq.kv8_compact(lq.Kv8Layers([cache]), _plan([context], [[-1] * 9], table=[[0, 1]], page=16), _i32([path]), _i32([kept]))
    torch.cuda.synchronize()
    return cache


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_compact_codes_stay_within_eight_bits(cuda_device, dim):
    # Scales of a few times the least 32-bit number: what the rows need, 180 / 127 and 300 / 127 of it, is rounded to one
    # and two of it, and codes of up to 180 and 150 times that would be needed: they stop at the ends, with their signs.
    rng = np.random.default_rng(dim)
    for old, new, scale in ((0, 3, 1), (1, 3, 1), (2, 5, 2)):
        codes = rng.integers(-60, 61, (2, 1, 16, dim)).astype(np.int8)
        codes[1, 0, 2, :2] = (60, -60)  # the row that moves: token 4 behind a context of 14
        cache = _two_pages(codes, np.array([[old * LEAST], [new * LEAST]], np.float32), 2, [0, 4])
        expect = np.clip(np.rint(codes[1, 0, 2].astype(np.float64) * (new / scale)), -128, 127)
        for got, got_scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            assert float(got_scale[0, 0]) == scale * LEAST
            assert np.array_equal(got[0, 0, 15].cpu().numpy(), expect)
            if old == scale:
                assert np.array_equal(got[0, 0, :15].cpu().numpy(), codes[0, 0, :15])
    # What needs less than half of the least number is zero.
    codes = rng.integers(-1, 2, (2, 1, 16, dim)).astype(np.int8)
    cache = _two_pages(codes, np.array([[0.0], [LEAST]], np.float32), 2, [0, 4])
    assert float(cache.k_scale[0, 0]) == 0.0 and torch.all(cache.k[0, 0, 15] == 0) and torch.all(cache.v[0, 0, 15] == 0)
    assert _status_ok()


@pytest.mark.parametrize("dim,page,kv,layers", [(32, 16, 2, 3), (64, 16, 3, 35), (96, 32, 1, 2), (128, 64, 2, 2), (64, 128, 1, 1)])
@pytest.mark.parametrize("ends", ["walk", "half", "last"])
def test_compact_codes_and_scales_are_the_definitions(cuda_device, dim, page, kv, layers, ends):
    rng = np.random.default_rng(dim + page + layers)
    sizes = [26, 0, 1, 2 * page + 9, 40, 300, 7]
    context = [0, 5, page - 1, page, 2 * page - 3, 301, 12]
    trees = [_random_tree(rng, n, "near") if n else [] for n in sizes]
    if ends == "walk":
        paths = [_path_of(t, int(rng.integers(0, len(t)))) if t else [] for t in trees]
    elif ends == "half":
        paths = [sorted(rng.choice(n, n // 2, replace=False).tolist()) for n in sizes]
    else:
        paths = [list(range(n // 2, n)) for n in sizes]
    lengths = [c + n for c, n in zip(context, sizes)]
    held = [ok.pages_of(n, page) for n in lengths]
    order, table, at = rng.permutation(sum(held) + 3), np.full((len(sizes), max(held) + 2), -1), 0
    for s, n in enumerate(held):
        table[s, :n] = order[at:at + n]
        at += n
    pool = order.size
    codes = rng.integers(-127, 128, (layers, 2, pool, kv, page, dim)).astype(np.int8)
    scales = (0.02 * np.exp(2.0 * rng.standard_normal((layers, 2, pool, kv)))).astype(np.float32)
    path = np.full((len(sizes), max(sizes)), -1)
    for s, way in enumerate(paths):
        path[s, :len(way)] = way
    kept = [len(p) for p in paths]
    caches = [lq.Kv8Cache(*(torch.from_numpy(c).cuda() for c in codes[i]), *(torch.from_numpy(x).cuda() for x in scales[i]))
              for i in range(layers)]
    lq.kv8_compact(lq.Kv8Layers(caches), _plan(context, trees, lengths=lengths, page=page, table=table), _i32(path), _i32(kept))
    grown = 0
    for i, cache in enumerate(caches):
        for side, got, got_scale in ((0, cache.k, cache.k_scale), (1, cache.v, cache.v_scale)):
            expect, expect_scale, _ = ok.compact(codes[i, side], scales[i, side], context, lengths, table, path, kept)
            assert np.array_equal(got_scale.cpu().numpy(), expect_scale)
            assert np.array_equal(got.cpu().numpy(), expect)
            grown += int((expect_scale != scales[i, side]).sum())
    assert grown > 0 or layers * kv == 1  # (of one layer and head, no page may need another scale)
    assert _status_ok()


# ------------------------------------------------------------- a run of them
class _Loop:
    """A serving loop's state and one step of it, of fixed bounds: 5 requests of at most 12 rows, 48 in all."""

    requests, rows, most, page, kv, group, dim, layers, vocab, pool = 5, 48, 12, 16, 2, 4, 64, 2, 6200, 10

    def __init__(self, order, rope):
        i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        self.context, self.taken, self.table, self.free = i(self.requests), i(1), i(self.requests, 12), _i32(order)
        self.new, self.ids, self.parents = i(self.requests), i(self.rows), i(self.rows)
        self.qkv, self.logits, self.probs = f(self.layers, self.rows, (self.group + 2) * self.kv * self.dim), f(self.rows, self.vocab), f(self.rows, self.vocab)
        self.accept, self.sample, self.heat = f(self.rows), f(self.requests), f(self.requests)
        self.caches = [lq.Kv8Cache(*(torch.zeros((self.pool, self.kv, self.page, self.dim), dtype=torch.int8, device="cuda") for _ in range(2)),
                                   *(torch.zeros((self.pool, self.kv), device="cuda") for _ in range(2))) for _ in range(self.layers)]
        self.stack, self.workspace, self.rope = lq.Kv8Layers(self.caches), lq.Kv8Workspace(), rope
        self.out = [f(self.rows, self.group * self.kv * self.dim) for _ in range(self.layers)]
        self.plan = self.tree = self.verdict = self.left = None

    def step(self):
        width = self.group * self.kv * self.dim
        self.plan = lq.kv8_plan(self.context, self.new, self.table, self.free, self.taken, self.page, self.rows, max_tokens=self.most, out=self.plan)
        self.tree = lq.kv8_tree(self.parents, self.plan, out=self.tree)
        for x, cache, out in zip(self.qkv, self.caches, self.out):
            lq.kv8_append(x[:, width:width + self.kv * self.dim], x[:, width + self.kv * self.dim:], cache, self.plan.slots, self.tree.positions, rope=self.rope)
            lq.kv8_tree_attention(x[:, :width], cache, self.plan, self.tree, self.dim ** -0.5, rope=self.rope, out=out, workspace=self.workspace)
        self.taken.copy_(self.plan.taken)
        self.verdict = lq.verify_drafts(self.logits, self.ids, self.parents, self.plan, self.accept, self.sample, self.heat, self.probs, out=self.verdict)
        lq.kv8_compact(self.stack, self.plan, self.verdict.path, self.verdict.kept)
        self.left = lq.kv8_release(self.plan, self.verdict.kept, self.free, self.taken, out=self.left)
        self.context.copy_(self.left.lengths)
        self.taken.copy_(self.left.taken)

    def state(self):
        return [self.context, self.taken, self.table, self.free, self.tree.positions, self.tree.masks, self.verdict.path, self.verdict.tokens,
                self.verdict.kept, self.verdict.next, *self.out, *(t for c in self.caches for t in (c.k, c.v, c.k_scale, c.v_scale))]


def test_a_captured_step_of_drafts_is_the_eager_one(cuda_device):
    # One graph over steps of unlike lengths and trees, some requests without rows, some refused when the pages run out.
    rng = np.random.default_rng(81)
    order, rope = rng.permutation(_Loop.pool), _rope_cuda(_rope(200, _Loop.dim))
    eager, graphed = _Loop(order, rope), _Loop(order, rope)
    graphed.step()  # of no tokens: the handles are made
    eager.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        graphed.step()
    drafted = refused = 0
    for step in range(24):
        new = rng.integers(0, _Loop.most + 1, _Loop.requests)
        while new.sum() > _Loop.rows:
            new[rng.integers(0, _Loop.requests)] = 0
        trees = [_random_tree(rng, int(n), "near") if n else [] for n in new]
        pad = _Loop.rows - int(new.sum())
        trees_in = trees if not pad else [*trees, [-1] * pad]  # (values for the rows behind the last)
        logits, ids, accept, sample, heat, q = _verify_case(rng, trees_in, _Loop.vocab, True)
        qkv = rng.standard_normal(eager.qkv.shape).astype(np.float32)
        accept *= 0.3
        for loop in (eager, graphed):
            for to, value in ((loop.new, new), (loop.ids, ids), (loop.parents, [p for t in trees_in for p in t])):
                to.copy_(_i32(value))
            for to, value in ((loop.logits, logits), (loop.probs, q), (loop.accept, accept), (loop.sample, sample[:5]), (loop.heat, heat[:5]), (loop.qkv, qkv)):
                to.copy_(_f32(value))
        before = eager.context.clone()
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), graphed.state()):
            assert torch.equal(a, b), step
        assert not torch.isnan(torch.stack(eager.out)[:, :int(new.sum())]).any()
        refused += int((eager.plan.lengths < before + eager.new).sum())
        drafted += int((eager.verdict.kept > 1).sum())
        held = [p for s in range(5) for p in eager.table[s, :ok.pages_of(int(eager.context[s]), _Loop.page)].tolist()]
        assert sorted(held + eager.free.tolist()[int(eager.taken):]) == list(range(_Loop.pool))
    assert drafted > 10 and refused > 0 and int(eager.context.max()) > _Loop.page
    assert _status_ok()
