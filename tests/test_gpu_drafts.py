"""The operators that check drafted tokens, on the GPU, against their definitions in
64-bit floats (oracle/kv8.py, oracle/drafts.py).

Tolerances, with u = 2^-24:
* trees, releases: whole numbers, equal.
* tree attention: as the causal one (test_gpu_kv8.py): |error| <= V * (2 (dim + 16) R + 64) u
  with the reach R of a row's scores and values up to V, and 1e-5 of the whole output's 2-norm.
* compaction: quotients and products in 64 bits (each off by at most 2^-53 of itself, three of
  them), so a code may differ by one where the exact number lies within 127 * 4 * 2^-53 of a
  half; a scale is rounded to 32 bits once, from a number within 2^-52 of the exact one, which
  may be the other of two neighbours: 2 u.
* verification: whole numbers, equal, where the oracle's nearest comparison is further from
  turning out the other way than the operator's own error: for a child 2^-17 of p (the
  exponentials' 32 bits: 2 ulp each and an exponent of up to 2^5 rounded to 2^-24 of itself,
  2^-18.5 at most), for a draw 2^-40 of the sum (64-bit sums of up to 2^20 terms, each of them
  within 2^-46).  Where a request is nearer than that it is left out, and at most 2 % may be.
"""
import numpy as np
import pytest
import torch

import leaf_b200 as lq
from leaf_b200 import _lib
from oracle import drafts as od
from oracle import kv8 as ok
from test_gpu_kv8 import U, _Batch, _i32, _rope_cuda, _status_ok

pytestmark = pytest.mark.gpu


def _f32(a):
    return torch.tensor(np.asarray(a), dtype=torch.float32, device="cuda")


def _prefix(x):
    return np.concatenate([[0], np.cumsum(np.asarray(x, dtype=np.int64))])


def _random_tree(rng, n, kind="near"):
    if kind == "chain":
        return [t - 1 for t in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "forest":
        return [-1 if t == 0 or rng.random() < 0.2 else int(rng.integers(0, t)) for t in range(n)]
    if kind == "binary":
        return [-1] + [(t - 1) // 2 for t in range(1, n)]
    return [-1] + [t - 1 - int((t - 1) * rng.random() ** 3) for t in range(1, n)]


def _plan(context, trees, pad=0, lengths=None, page=None, table=None, most=None):
    new = [len(p) for p in trees]
    lengths = [c + n for c, n in zip(context, new)] if lengths is None else lengths
    table = np.zeros((len(trees), 1)) if table is None else table
    return lq.Kv8Plan(_i32(context), _i32(lengths), _i32(_prefix(new)), _i32(np.zeros(len(trees) + 1)), _i32(table),
                      sum(new) + pad, max(new, default=0) if most is None else most, page=page)


# ------------------------------------------------------------------- trees
def _check_tree(context, trees, pad=0, words=None):
    plan = _plan(context, trees, pad)
    parents = _i32([p for t in trees for p in t] + [0] * pad)
    if words is None:
        got = lq.kv8_tree(parents, plan)
    else:
        got = lq.Kv8Tree(torch.full((plan.tokens,), 7, dtype=torch.int32, device="cuda"),
                         torch.full((plan.tokens, words), 7, dtype=torch.int32, device="cuda"))
        assert lq.kv8_tree(parents, plan, out=got) is got
    positions, masks = got.positions.tolist(), got.masks.cpu().numpy().view(np.uint32)
    at = 0
    for c, parents in zip(context, trees):
        expect, above = ok.tree(parents, c)
        assert positions[at:at + len(parents)] == expect
        for t, row in enumerate(above):
            bits = sum(1 << i for i in row)
            assert [int(w) for w in masks[at + t]] == [bits >> 32 * w & 0xffffffff for w in range(masks.shape[1])]
        at += len(parents)
    assert positions[at:] == [-1] * pad and not masks[at:].any()
    return got


@pytest.mark.parametrize("kind", ["near", "chain", "star", "forest", "binary"])
@pytest.mark.parametrize("sizes", [[1], [2, 0, 31], [32, 33, 1, 64, 65], [26] * 64, [300, 7, 255, 0, 256], [1024, 1, 1023]])
def test_tree(cuda_device, kind, sizes):
    rng = np.random.default_rng(len(sizes) + sum(sizes))
    context = rng.integers(0, 5000, len(sizes))
    trees = [_random_tree(rng, n, kind) if n else [] for n in sizes]
    _check_tree(context, trees)
    _check_tree(context, trees, pad=13)
    if max(sizes) <= 64:
        _check_tree(context, trees, pad=2, words=32)
    assert _status_ok()


def test_tree_broken_parents_empty_their_rows(cuda_device):
    # A parent that is no earlier row: itself, a later one, past the tree, below -1; and the rows behind it.
    for bad in (3, 4, 9, 2**31 - 1, -2, -2**31):
        trees = [[-1, 0, 1, bad, 3, 4, 2, -1], [-1, 0]]
        _check_tree([5, 70], trees)
        assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    chain = [t - 1 for t in range(200)]
    chain[40] = 40  # the way of rows in later words
    _check_tree([0], [chain])
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    assert _status_ok()


def test_tree_of_no_tokens_and_of_too_many(cuda_device):
    plan = _plan([4, 5], [[], []])
    assert lq.kv8_tree(_i32([]), plan).positions.numel() == 0
    # More rows than the bound says: the others see nothing, and it is reported.
    plan = _plan([4], [[-1, 0, 1, 2]], most=2)
    got = lq.kv8_tree(_i32([-1, 0, 1, 2]), plan)
    assert got.positions.tolist() == [4, 5, -1, -1] and got.masks.tolist() == [[1], [3], [0], [0]]
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID


# --------------------------------------------------------------- attention
class _Trees(_Batch):
    """A step of trees over random caches."""

    def __init__(self, rng, context, new, *args, kind="near", **more):
        super().__init__(rng, context, new, *args, **more)
        self.trees = [_random_tree(rng, n, kind) if n else [] for n in new]
        self.pad = self.tokens - sum(new)
        self.parents = _i32([p for t in self.trees for p in t] + [0] * self.pad)
        self.tree = lq.kv8_tree(self.parents, self.plan)

    def run(self, q=None, **more):
        q = torch.from_numpy(self.q).cuda() if q is None else q
        return lq.kv8_tree_attention(q, self.cache, self.plan, self.tree, self.scale, rope=_rope_cuda(self.rope), **more)

    def check(self, got=None):
        got = (self.run() if got is None else got).cpu().numpy().astype(np.float64)
        expect, bound = np.zeros_like(got), np.zeros_like(got)
        heads, at = self.kv * self.group, 0
        for s, (c, n) in enumerate(zip(self.context, self.new)):
            positions, above = ok.tree(self.trees[s], c)
            q = ok.rotate(self.q[at:at + n].reshape(n, heads, self.dim), np.maximum(np.array(positions, dtype=int), 0), self.rope)
            held = self.table[s, :ok.pages_of(self.lengths[s], self.page)]
            visible = np.zeros((n, held.size * self.page), dtype=bool)
            for t, rows in enumerate(above):
                if rows:
                    visible[t, :min(c, self.lengths[s])] = True
                    visible[t, [c + i for i in rows if c + i < self.lengths[s]]] = True
            for h in range(self.kv):
                k, v = (self.codes[i][held, h].reshape(-1, self.dim).astype(np.float64) *
                        np.repeat(self.scales[i][held, h].astype(np.float64), self.page)[:, None] for i in range(2))
                out, reach = ok.tree_attention(q[:, h * self.group:(h + 1) * self.group], visible, k, v, self.scale)
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
@pytest.mark.parametrize("group", [1, 2, 3, 8, 12])
def test_tree_attention_few_rows(cuda_device, dim, group):
    rng = np.random.default_rng(dim + group)
    _Trees(rng, [0, 1, 15, 63, 64, 300], [1, 2, 3, 5, 7, 9], 64, 2, group, dim, rotary=dim).check()
    _Trees(rng, [0, 33, 200], [5, 0, 6], 16, 1, group, dim, kind="forest").check()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kind", ["near", "chain", "star", "forest", "binary"])
def test_tree_attention_pages_and_shapes(cuda_device, page, kind):
    rng = np.random.default_rng(page)
    context = [0, 1, page - 1, page, page + 1, 3 * page - 5, 700, 17]
    _Trees(rng, context, [12, 0, 1, 40, 33, 31, 7, 64], page, 3, 4, 64, rotary=32, kind=kind).check()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("kv,group,page", [(32, 1, 64), (12, 3, 16), (8, 8, 64), (4, 16, 128), (13, 5, 32)])
def test_tree_attention_many_rows(cuda_device, dim, kv, group, page):
    # Enough query rows for the kernel that tiles them by 128.
    rng = np.random.default_rng(dim + kv + page)
    _Trees(rng, [0, 300, 95, 0, 17], [97, 1, 33, 0, 64], page, kv, group, dim, rotary=dim // 2).check()
    _Trees(rng, [200, 31], [60, 70], page, kv, group, dim, rotary=dim, kind="forest").check()


@pytest.mark.parametrize("new", [40, 95, 96, 97, 193])
@pytest.mark.parametrize("kind", ["near", "star", "forest"])
def test_tree_attention_tile_edges(cuda_device, new, kind):
    rng = np.random.default_rng(new)
    _Trees(rng, [0, 96 - new % 96], [new, new], 16, 16, 4, 64, rotary=64, kind=kind).check()
    _Trees(rng, [64, 500], [new, 1], 128, 16, 6, 128, kind=kind).check()


def test_tree_attention_long_caches_and_large_trees(cuda_device):
    rng = np.random.default_rng(21)
    _Trees(rng, [20000, 3, 9001], [26, 4, 13], 128, 2, 8, 64, rotary=64).check()      # parts joined
    _Trees(rng, [12000], [60], 32, 4, 16, 64, kind="forest").check()                  # tiles in parts
    _Trees(rng, [100, 0], [1024, 1000], 64, 2, 2, 64, rotary=64).check()
    _Trees(rng, [50], [1024], 64, 1, 1, 32, kind="binary").check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("context,requests,new", [(2900, 1, 64), (2900, 1, 33), (2100, 4, 16), (1500, 2, 64), (700, 1, 128)])
def test_tree_attention_few_items(cuda_device, dim, context, requests, new):
    # 2,048 rows and more, fewer items than blocks: short ones are cut and joined, at 2,048 keys' room too.
    rng = np.random.default_rng(context + new + dim)
    _Trees(rng, [context] * requests, [new] * requests, 64, 8, 4, dim, rotary=dim).check()
    _Trees(rng, [context, 0, 40][:requests + 2], [new, 1, 7], 16, 8, 8, dim, kind="binary").check()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_tree_attention_items_that_leave_a_half_without_keys(cuda_device, dim):
    # 264 rows a head: an item of both halves, then one of 8 rows whose only tile the first half has.
    rng = np.random.default_rng(dim)
    _Trees(rng, rng.integers(0, 25, 200), [33] * 200, 64, 2, 8, dim, rotary=dim).check()
    # The same of parts: items of several tiles, cut into shares.
    _Trees(rng, rng.integers(0, 800, 60), [*rng.integers(1, 34, 59), 33], 16, 1, 16, dim).check()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("wide", [9, 12, 16])
def test_tree_attention_items_of_one_half_behind_those_of_both(cuda_device, dim, wide):
    # Of 144 to 256 rows and one tile, the second half's fewer; then of 96 rows and two, whose keys the halves share.
    rng = np.random.default_rng(dim + wide)
    _Trees(rng, [30, 97] * 90, [wide, 6] * 90, 16, 2, 16, dim, rotary=dim).check()


@pytest.mark.parametrize("requests", [200, 500])
def test_tree_attention_many_requests(cuda_device, requests):
    rng = np.random.default_rng(requests)
    _Trees(rng, rng.integers(0, 200, requests), rng.integers(0, 6, requests), 16, 2, 2, 64, rotary=64).check()


@pytest.mark.parametrize("new,kv,group", [(6, 2, 4), (60, 8, 8)])
def test_tree_attention_of_a_chain_is_the_causal_one(cuda_device, new, kv, group):
    rng = np.random.default_rng(new)
    b = _Trees(rng, [130, 0, 64], [new] * 3, 32, kv, group, 64, rotary=64, kind="chain")
    tree, causal = b.run(), _Batch.run(b)  # each within about 1e-6 of the exact one
    assert torch.linalg.norm(tree - causal) <= 2e-6 * torch.linalg.norm(causal)


@pytest.mark.parametrize("new,kv,group", [(6, 2, 4), (60, 8, 8)])
@pytest.mark.parametrize("rotary", [0, 64])
def test_tree_attention_rows_that_see_nothing(cuda_device, new, kv, group, rotary):
    # Rows that hang from nowhere give zeros, refused requests see their cached tokens only, rows past the last stay.
    rng = np.random.default_rng(34)
    b = _Trees(rng, [0, 20, 64, 0], [new] * 4, 16, kv, group, 64, lengths=[0, 20, 64 + new, 0], spare=40, pad=2, rotary=rotary)
    b.trees[2][3] = 3
    b.parents = _i32([p for t in b.trees for p in t] + [0, 0])
    b.tree = lq.kv8_tree(b.parents, b.plan)
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    b.q[-2:] = np.nan
    out = b.run(out=torch.full(b.q.shape, 7.0, device="cuda"))
    empty = [t for t, rows in enumerate(ok.tree(b.trees[2], 64)[1]) if not rows]
    assert torch.all(out[:new] == 0) and torch.all(out[3 * new:4 * new] == 0) and torch.all(out[-2:] == 7.0)
    assert empty and torch.all(out[[2 * new + t for t in empty]] == 0)
    b.check(out)


@pytest.mark.parametrize("new,kv,group", [(6, 2, 4), (60, 8, 8)])
def test_tree_attention_stays_clear_of_what_a_row_does_not_see(cuda_device, new, kv, group):
    # A page of drafts whose scales are no numbers shows in the rows that see one of them, and in no others.
    rng = np.random.default_rng(35)
    b = _Trees(rng, [16], [new], 16, kv, group, 64, kind="star", spare=8)
    page = (16 + new - 1) // 16
    first = page * 16 - 16
    for which in (0, 1):
        b.scales[which][b.table[0, page]] = np.nan
    b.cache.k_scale.copy_(torch.from_numpy(b.scales[0]))
    b.cache.v_scale.copy_(torch.from_numpy(b.scales[1]))
    out = b.run()
    sees = [any(i >= first for i in rows) for rows in ok.tree(b.trees[0], 16)[1]]
    for t, s in enumerate(sees):
        assert torch.isnan(out[t]).all() if s else torch.isfinite(out[t]).all()
    assert any(sees)
    if not all(sees):
        keep = [t for t, s in enumerate(sees) if not s]
        assert torch.all(out[keep].abs() < 10)
    # Scores that stand far above: of the keys that a row does not see.
    b.scales[:, b.table[0, page]] = 0.03
    b.scales[0, b.table[0, page]] = 2000.0
    b.cache.k_scale.copy_(torch.from_numpy(b.scales[0]))
    b.cache.v_scale.copy_(torch.from_numpy(b.scales[1]))
    clear = b.run()
    keep = [t for t, s in enumerate(sees) if not s]
    b.scales[0, b.table[0, page]] = 0.02
    b.cache.k_scale.copy_(torch.from_numpy(b.scales[0]))
    quiet = b.run()
    scale = quiet[keep].abs().amax() if keep else 0
    assert not keep or torch.all((clear[keep] - quiet[keep]).abs() <= 1e-5 * scale)
    assert _status_ok()


def test_tree_attention_reports_positions_and_pages(cuda_device):
    rng = np.random.default_rng(36)
    for new, kv, group in ((6, 2, 4), (60, 8, 8)):
        b = _Trees(rng, [30], [new], 16, kv, group, 64, rotary=64, kind="star", spare=4)
        b.tree.positions[2] = b.rope[0].shape[0] + 5
        out = b.run()
        assert torch.all(out[2] == 0) and torch.isfinite(out).all()
        assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
        b.tree.positions[2] = 31
        b.plan.table[0, 0] = b.pool
        assert torch.isfinite(b.run()).all()
        assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    assert _status_ok()


def test_tree_attention_strides_streams_graphs_and_workspaces(cuda_device):
    rng = np.random.default_rng(37)
    small = _Trees(rng, [100, 40], [5, 9], 16, 2, 4, 64, rotary=64)
    large = _Trees(rng, [100, 40], [70, 60], 16, 8, 8, 64, rotary=64)
    workspace = lq.Kv8Workspace()
    expect = [small.run(), large.run()]
    # Columns of a wider matrix, one workspace for both forms and for causal calls in between.
    for _ in range(2):
        for b, e in zip((small, large), expect):
            wide = torch.full((b.tokens, b.q.shape[1] + 64), np.nan, device="cuda")
            wide[:, :-64] = torch.from_numpy(b.q).cuda()
            assert torch.equal(b.run(wide[:, :-64], workspace=workspace), e)
            _Batch.run(b, workspace=workspace)
    side = torch.cuda.Stream()
    q = [torch.from_numpy(b.q).cuda() for b in (small, large)]
    rope = [_rope_cuda(b.rope) for b in (small, large)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = [lq.kv8_tree_attention(x, b.cache, b.plan, b.tree, b.scale, rope=r, workspace=workspace)
               for x, b, r in zip(q, (small, large), rope)]
    side.synchronize()
    assert all(torch.equal(o, e) for o, e in zip(out, expect))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for b, x, r, o in zip((small, large), q, rope, out):
            lq.kv8_tree(b.parents, b.plan, out=b.tree)
            lq.kv8_tree_attention(x, b.cache, b.plan, b.tree, b.scale, rope=r, out=o, workspace=workspace)
    for o in out:
        o.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, e) for o, e in zip(out, expect))
    assert _status_ok()


# ----------------------------------------------------------------- compact
def _path_of(parents, end):
    way = []
    while end >= 0:
        way.append(end)
        end = parents[end]
    return way[::-1]


def _check_compact(rng, context, sizes, page, kv, dim, layers, kind="near", paths=None, lengths=None, spread=0.5, kept=None):
    trees = [_random_tree(rng, n, kind) if n else [] for n in sizes]
    lengths = [c + n for c, n in zip(context, sizes)] if lengths is None else lengths
    if paths is None:
        paths = [_path_of(p, int(rng.integers(0, len(p)))) if p else [] for p in trees]
    width = max(sizes)
    held = [ok.pages_of(n, page) for n in lengths]
    pool = sum(held) + 2
    order = rng.permutation(pool)
    table, at = np.full((len(sizes), max(held) + 1), -1), 0
    for s, b in enumerate(held):
        table[s, :b] = order[at:at + b]
        at += b
    codes = np.clip(np.rint(rng.standard_normal((layers, 2, pool, kv, page, dim)) * 38), -127, 127).astype(np.int8)
    scales = (0.02 * np.exp(spread * rng.standard_normal((layers, 2, pool, kv)))).astype(np.float32)
    path = np.full((len(sizes), width), -1)
    for s, way in enumerate(paths):
        path[s, :len(way)] = way
    kept = [len(p) for p in paths] if kept is None else kept
    caches = [lq.Kv8Cache(*(torch.from_numpy(c).cuda() for c in codes[i]), *(torch.from_numpy(x).cuda() for x in scales[i]))
              for i in range(layers)]
    plan = _plan(context, trees, lengths=lengths, page=page, table=table)
    lq.kv8_compact(lq.Kv8Layers(caches), plan, _i32(path), _i32(kept))
    torch.cuda.synchronize()
    grown = moved = 0
    for i, cache in enumerate(caches):
        for side, got, got_scale in ((0, cache.k, cache.k_scale), (1, cache.v, cache.v_scale)):
            expect, expect_scale, unrounded = ok.compact(codes[i, side], scales[i, side], context, lengths, table, path, kept)
            got, got_scale = got.cpu().numpy(), got_scale.cpu().numpy()
            assert np.all(np.abs(got_scale - expect_scale) <= 2 * U * expect_scale)
            grown += int((expect_scale != scales[i, side]).sum())
            moved += int((expect != codes[i, side]).sum())
            if np.array_equal(got_scale, expect_scale):
                tie = np.abs(np.abs(unrounded - np.floor(unrounded)) - 0.5) < 127 * 4 * 2.0 ** -53
                differ = got != expect
                assert not np.any(differ & ~tie), f"{int((differ & ~tie).sum())} codes differ"
            assert np.all(np.abs(got.astype(int) - expect) <= 1)
    return grown, moved


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_compact_pages_and_heads(cuda_device, dim, page):
    rng = np.random.default_rng(dim + page)
    context = [0, 1, page - 1, page, 2 * page - 3, 300, 5]
    _, moved = _check_compact(rng, context, [26, 1, 40, 2 * page + 5, 0, 200, 9], page, 3, dim, 2)
    assert moved > 0
    assert _status_ok()


@pytest.mark.parametrize("kind", ["near", "chain", "star", "binary"])
@pytest.mark.parametrize("layers", [1, 22, 33, 70])
def test_compact_layers_and_shapes(cuda_device, kind, layers):
    rng = np.random.default_rng(layers)
    sizes = rng.integers(0, 40, 9)
    sizes[0] = 40
    grown, moved = _check_compact(rng, rng.integers(0, 100, 9), sizes, 16, 2, 32, layers, kind=kind)
    assert (moved > 0) == (kind != "chain")
    assert _status_ok()


def test_compact_long_paths(cuda_device):
    rng = np.random.default_rng(3)
    for sizes, context in (([1024, 700], [77, 0]), ([500], [15])):
        paths = [sorted(rng.choice(n, n // 2, replace=False).tolist()) for n in sizes]
        grown, _ = _check_compact(rng, context, sizes, 16, 2, 64, 1, paths=paths)
        assert grown > 0  # rows of one page out of two, each with a scale of its own
        _check_compact(rng, context, sizes, 128, 1, 128, 2, paths=paths, spread=2.0)
        _check_compact(rng, context, sizes, 64, 1, 96, 1, paths=[list(range(n // 2, n)) for n in sizes])
        _check_compact(rng, context, sizes, 64, 1, 96, 1, paths=[[0] + list(range(2, n)) for n in sizes])
    assert _status_ok()


def test_compact_many_requests(cuda_device):
    rng = np.random.default_rng(4)
    _check_compact(rng, rng.integers(0, 60, 700), rng.integers(0, 12, 700), 16, 1, 32, 2)
    assert _status_ok()


def test_compact_bounds(cuda_device):
    # More kept than there are rows, or than fit the path; requests that were refused; none kept, and fewer than none.
    rng = np.random.default_rng(5)
    _check_compact(rng, [10, 4, 7, 30, 2], [9, 9, 9, 9, 9], 16, 2, 64, 2, paths=[[0, 3, 8]] * 5, kept=[3, 1, 0, -4, 2],
                   lengths=[19, 13, 16, 30, 11])
    _check_compact(rng, [10], [9], 16, 2, 64, 1, paths=[[0, 2, 3, 4, 5, 6, 7, 8]], kept=[8])
    _check_compact(rng, [10, 8], [4, 4], 16, 1, 64, 1, paths=[[1, 2, 3], [0, 1, 2, 3]], kept=[3, 2**31 - 1])
    assert _status_ok()


@pytest.mark.parametrize("bad", [[0, 2, 2], [0, 4, 3], [3, 1, 2], [0, 9, 10], [0, 5, -1], [0, -7, 5], [2**31 - 1, 1, 2]])
def test_compact_leaves_requests_with_a_broken_path(cuda_device, bad):
    rng = np.random.default_rng(6)
    _check_compact(rng, [10, 20], [9, 9], 16, 2, 64, 2, paths=[[0, 4, 6], bad])
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID


def test_compact_leaves_requests_with_pages_outside_the_pool(cuda_device):
    rng = np.random.default_rng(7)
    for bad in (-1, 6, 2**31 - 1, -2**31):
        codes = rng.integers(-127, 128, (2, 6, 1, 16, 32)).astype(np.int8)
        scales = np.full((2, 6, 1), 0.1, np.float32)
        for broken in (0, 1):  # where the row comes from, and where it goes
            cache = lq.Kv8Cache(*(torch.from_numpy(c).cuda() for c in codes), *(torch.from_numpy(s).cuda() for s in scales))
            table = np.array([[0, 1], [2, 3]])
            table[1, 1 - broken] = bad
            plan = _plan([14, 14], [[-1] * 5] * 2, table=table, page=16)
            lq.kv8_compact(lq.Kv8Layers([cache]), plan, _i32([[0, 4], [1, 4]]), _i32([2, 2]))
            torch.cuda.synchronize()
            assert torch.equal(cache.k[2:].cpu(), torch.from_numpy(codes[0, 2:]))
            assert torch.equal(cache.k[0, 0, 15].cpu(), torch.from_numpy(codes[0, 1, 0, 2]))
            assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    # A request whose length does not fit its row of the table.
    plan = _plan([40], [[-1] * 5], table=[[0, 1]], page=16)
    before = cache.k.clone()
    lq.kv8_compact(lq.Kv8Layers([cache]), plan, _i32([[0, 4]]), _i32([2]))
    assert torch.equal(cache.k, before) and _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID


def test_compact_scales_that_are_no_numbers_and_zeros(cuda_device):
    def case(old, new):
        codes = torch.arange(1, 1 + 3 * 16 * 32, device="cuda").remainder(200).sub(100).to(torch.int8).reshape(3, 1, 16, 32)
        scales = torch.tensor([[old], [new], [1.0]], device="cuda")
        cache = lq.Kv8Cache(codes.clone(), codes.clone(), scales, scales.clone())
        lq.kv8_compact(lq.Kv8Layers([cache]), _plan([14], [[-1] * 9], table=[[0, 1]], page=16), _i32([[0, 4]]), _i32([2]))
        torch.cuda.synchronize()
        return codes, cache

    nan, inf = float("nan"), float("inf")
    codes, cache = case(0.5, nan)
    assert torch.isnan(cache.k_scale[0, 0])  # the page shows what went in
    codes, cache = case(nan, 0.5)
    assert torch.isnan(cache.k_scale[0, 0]) and torch.equal(cache.k[0, 0, :15], codes[0, 0, :15])
    codes, cache = case(nan, nan)
    assert torch.isnan(cache.k_scale[0, 0]) and torch.equal(cache.k[0, 0, 15], codes[1, 0, 2])
    codes, cache = case(0.5, inf)
    assert torch.isinf(cache.k_scale[0, 0]) and torch.all(cache.k[0, 0, :15] == 0)
    codes, cache = case(0.0, 0.0)
    assert float(cache.k_scale[0, 0]) == 0.0 and torch.equal(cache.k[0, 0, 15], codes[1, 0, 2])
    codes, cache = case(0.5, 0.0)
    assert float(cache.k_scale[0, 0]) == 0.5 and torch.all(cache.k[0, 0, 15] == 0)
    assert torch.equal(cache.k[1:], codes[1:]) and torch.equal(cache.k[0, 0, :15], codes[0, 0, :15])
    assert _status_ok()


# ----------------------------------------------------------------- release
def _check_release(context, lengths, kept, table, free, taken, page, out=None):
    expect, expect_free, expect_taken = ok.release(context, lengths, kept, table, free, taken, page)
    plan = lq.Kv8Plan(_i32(context), _i32(lengths), _i32(np.zeros(len(context) + 1)), _i32(np.zeros(len(context) + 1)),
                      _i32(table), 0, 0, page=page)
    pages = _i32(free)
    got = lq.kv8_release(plan, _i32(kept), pages, _i32([taken]), out=out)
    torch.cuda.synchronize()
    assert got.lengths.tolist() == expect.tolist() and int(got.taken) == expect_taken
    assert pages.tolist() == expect_free.tolist()
    return got


def _release_case(rng, requests, page, longest, most):
    context = rng.integers(0, longest + 1, requests)
    fresh = rng.integers(0, most + 1, requests)
    lengths = context + fresh
    held = [ok.pages_of(int(n), page) for n in lengths]
    order = rng.permutation(sum(held) + 50)
    table, at = np.full((requests, max(held, default=0) + 1), -1), 0
    for s, b in enumerate(held):
        table[s, :b] = order[at:at + b]
        at += b
    kept = np.array([int(rng.integers(0, f + 1)) for f in fresh])
    return context, lengths, kept, table, order, at


@pytest.mark.parametrize("requests", [1, 3, 64, 256, 257, 1025, 2500])
@pytest.mark.parametrize("page,longest,most", [(16, 40, 1), (16, 300, 70), (64, 500, 200), (128, 1000, 3)])
def test_release(cuda_device, requests, page, longest, most):
    rng = np.random.default_rng(requests * 100 + page + most)
    context, lengths, kept, table, free, taken = _release_case(rng, requests, page, longest, most)
    got = _check_release(context, lengths, kept, table, free, taken, page)
    ends = np.where(rng.random(requests) < 0.3, -context, kept)  # some requests end
    ends[rng.random(requests) < 0.1] = -2**31
    ends[rng.random(requests) < 0.1] = 2**31 - 1
    _check_release(context, lengths, ends, table, free, taken, page, out=got)
    _check_release(context, lengths, -context, table, free, taken, page)  # all do
    assert _status_ok()


def test_release_refuses_what_does_not_fit(cuda_device):
    rng = np.random.default_rng(8)
    for requests in (5, 400, 1500):
        context, lengths, kept, table, free, taken = _release_case(rng, requests, 16, 100, 60)
        for low in (0, 1, 5):
            _check_release(context, lengths, -context, table, free, low, 16)
            assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
        _check_release(context, lengths, -context, table, free[:taken - 1], taken, 16)
        assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    # Lengths that are none, or do not fit the table's row, are kept.
    plan = lq.Kv8Plan(_i32([3, 3, 3]), _i32([-5, 33, 32]), _i32([0] * 4), _i32([0] * 4), _i32([[0, 1], [2, 3], [4, 5]]), 0, 0, page=16)
    free = _i32([9, 9, 9, 9])
    got = lq.kv8_release(plan, _i32([0, 0, 0]), free, _i32([4]))
    assert got.lengths.tolist() == [-5, 33, 3] and int(got.taken) == 3 and free.tolist() == [9, 9, 9, 5]
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    assert _status_ok()


def test_release_of_nothing(cuda_device):
    _check_release([], [], [], np.zeros((0, 3)), [1, 2], 1, 64)
    _check_release([5, 0], [5, 0], [0, 0], [[0], [1]], [], 0, 64)
    assert _status_ok()


def test_plan_and_release_keep_every_page_once(cuda_device):
    # Twenty steps that take pages and give some back: no page is ever held twice.
    rng = np.random.default_rng(9)
    requests, page = 30, 16
    free, taken = _i32(rng.permutation(400)), _i32([0])
    table, length = _i32(np.full((requests, 40), -1)), _i32(np.zeros(requests))
    plan = left = None
    for step in range(20):
        new = rng.integers(0, 25, requests)
        plan = lq.kv8_plan(length, _i32(new), table, free, taken, page, 800, out=plan)
        kept = np.where(rng.random(requests) < 0.2, -1000, rng.integers(0, new + 1))
        left = lq.kv8_release(plan, _i32(kept), free, plan.taken, out=left)
        length.copy_(left.lengths)
        taken.copy_(left.taken)
        held = [p for s in range(requests) for p in table[s, :ok.pages_of(int(length[s]), page)].tolist()]
        rest = free.tolist()[int(taken):]
        assert sorted(held + rest) == list(range(400))
    assert _status_ok()


# ------------------------------------------------------------ verification
def _verify_case(rng, trees, vocab, probs, greedy=0.0, stride=0):
    tokens = sum(map(len, trees))
    logits = (rng.standard_normal((tokens, vocab)) * 4).astype(np.float32)
    drafted = logits + rng.standard_normal((tokens, vocab)).astype(np.float32)
    q = np.exp(drafted - drafted.max(axis=1, keepdims=True)).astype(np.float64)
    q = (q / q.sum(axis=1, keepdims=True)).astype(np.float32) if probs else None
    ids, at = [], 0
    for parents in trees:
        rank = {}
        for t, p in enumerate(parents):
            row = at + max(p, 0)
            rank[p] = rank.get(p, -1) + 1
            if probs:
                ids.append(int(rng.choice(vocab, p=q[row].astype(np.float64) / q[row].astype(np.float64).sum())))
            else:
                ids.append(int(np.argsort(-drafted[row])[min(rank[p], vocab - 1)]))
        at += len(parents)
    heat = rng.uniform(0.5, 1.5, len(trees))
    heat[rng.random(len(trees)) < greedy] = 0.0
    return logits, np.array(ids, dtype=np.int64), rng.random(tokens).astype(np.float32), rng.random(len(trees)).astype(np.float32), \
        heat.astype(np.float32), q


def _check_verify(trees, logits, ids, accept, sample, heat, q, pad=0, strided=0, most=None, out=None):
    new = [len(p) for p in trees]
    tokens, vocab = logits.shape
    plan = _plan([0] * len(trees), trees, pad=pad, most=most)
    more = lambda x, fill: np.concatenate([x, np.full((pad, *x.shape[1:]), fill, x.dtype)])  # noqa: E731
    dev = lambda x: _f32(more(x, np.nan))  # noqa: E731
    if strided:
        dev = lambda x: torch.cat((_f32(more(x, np.nan)), torch.full((tokens + pad, strided), float("nan"), device="cuda")),  # noqa: E731
                                  dim=1)[:, :vocab]
    parents = [p for t in trees for p in t]
    got = lq.verify_drafts(dev(logits), _i32(list(ids) + [0] * pad), _i32(parents + [0] * pad), plan, _f32(more(accept, 0.5)),
                           _f32(sample), _f32(heat), draft_probs=None if q is None else dev(q), out=out)
    torch.cuda.synchronize()
    path, toks, kept, nxt = (t.cpu().numpy() for t in (got.path, got.tokens, got.kept, got.next))
    at, near = 0, 0
    for s, p in enumerate(trees):
        rows = slice(at, at + new[s])
        way, tokens_out, (child, draw) = od.verify(logits[rows], ids[rows], p, accept[rows], sample[s], heat[s], None if q is None else q[rows])
        at += new[s]
        assert np.all(path[s, kept[s]:] == -1) and np.all(toks[s, kept[s]:] == -1)
        if child < 2.0 ** -17 or draw < 2.0 ** -40:
            near += 1
            continue
        assert kept[s] == len(way) and path[s, :kept[s]].tolist() == way
        assert toks[s, :kept[s]].tolist() == tokens_out and nxt[s] == (tokens_out[-1] if way else -1)
    assert near <= max(1, 0.02 * len(trees))
    return got


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 33, 500, 4099, 32000])
def test_verify_vocabularies(cuda_device, probs, vocab):
    rng = np.random.default_rng(vocab)
    trees = [_random_tree(rng, n, k) if n else [] for n, k in ((5, "chain"), (0, ""), (7, "binary"), (1, "near"), (9, "star"), (12, "near"))]
    _check_verify(trees, *_verify_case(rng, trees, vocab, probs))
    _check_verify(trees, *_verify_case(rng, trees, vocab, probs, greedy=0.5), pad=3, strided=5)
    assert _status_ok()


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("requests", [1, 17, 36, 70, 140, 400])
def test_verify_batches(cuda_device, probs, requests):
    # From eight blocks a request to one.
    rng = np.random.default_rng(requests)
    trees = [_random_tree(rng, int(n), "near") if n else [] for n in rng.integers(0, 8, requests)]
    trees[0] = _random_tree(rng, 6, "binary")
    _check_verify(trees, *_verify_case(rng, trees, 801, probs, greedy=0.2))
    assert _status_ok()


@pytest.mark.parametrize("probs", [False, True])
def test_verify_draws_where_the_sum_says(cuda_device, probs):
    # Every border of a row's sum, from both sides: numbers of 2^-10 of each other are exact.
    vocab, requests = 64, 400
    rng = np.random.default_rng(3)
    sample = np.concatenate([np.arange(requests - 3) / (requests - 3), [0.0, 1 - 2.0 ** -24, 0.5]]).astype(np.float32)
    trees = [[-1, 0]] * requests
    logits = np.repeat(rng.standard_normal((requests, vocab)).astype(np.float32) * 3, 2, axis=0)
    q = np.full((2 * requests, vocab), 1 / vocab, np.float32) if probs else None
    ids = np.repeat(rng.integers(0, vocab, requests), 2)
    accept = np.full(2 * requests, 0.999, np.float32)
    _check_verify(trees, logits, ids, accept, sample, np.full(requests, 0.9, np.float32), q)
    # Equal logits: token j for sample in [j / 64, (j + 1) / 64), the ends included on the left.
    flat = np.zeros((64, 64), np.float32)
    got = lq.verify_drafts(_f32(flat), _i32([0] * 64), _i32([-1] * 64), _plan([0] * 64, [[-1]] * 64), _f32(np.zeros(64)),
                           _f32(np.arange(64) / 64), _f32(np.ones(64)))
    assert got.next.tolist() == list(range(64))
    got = lq.verify_drafts(_f32(flat), _i32([0] * 64), _i32([-1] * 64), _plan([0] * 64, [[-1]] * 64), _f32(np.zeros(64)),
                           _f32(np.nextafter(np.float32(np.arange(1, 65) / 64), np.float32(0))), _f32(np.ones(64)))
    assert got.next.tolist() == list(range(64))


def test_verify_greedy_takes_the_first_of_the_largest(cuda_device):
    logits = np.zeros((6, 1000), np.float32)
    for row, (a, b) in enumerate(((999, 3), (17, 400), (0, 999), (128, 129), (500, 2), (77, 78))):
        logits[row, [a, b]] = 5.0
    # row 0's first largest is 3, row 1's 17, row 2's 0
    parents, ids = [-1, 0, 0, 2, 3, 3], [8, 999, 3, 0, 5, 128]
    got = lq.verify_drafts(_f32(logits), _i32(ids), _i32(parents), _plan([0], [parents]), _f32([np.nan] * 6), _f32([np.nan]),
                           _f32([0.0]))
    assert got.path.tolist() == [[0, 2, 3, 5, -1, -1]] and got.tokens.tolist() == [[3, 0, 128, 77, -1, -1]]
    assert got.kept.tolist() == [4] and got.next.tolist() == [77]
    for heat in (-1.0, float("nan"), -0.0):
        again = lq.verify_drafts(_f32(logits), _i32(ids), _i32(parents), _plan([0], [parents]), _f32([0.0] * 6), _f32([0.0]),
                                 _f32([heat]))
        assert torch.equal(again.path, got.path) and torch.equal(again.tokens, got.tokens)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_siblings_of_the_same_token(cuda_device, probs):
    # The same draft twice (and more): the second has what the first left.
    rng = np.random.default_rng(4)
    requests, vocab, n = 300, 11, 40
    parents = [-1] + [0] * (n - 1)
    trees = [parents] * requests
    logits, _, accept, sample, heat, q = _verify_case(rng, trees, vocab, probs)
    ids = rng.integers(0, vocab, requests * n)
    accept = rng.uniform(0.7, 1.0, accept.shape).astype(np.float32)
    _check_verify(trees, logits, ids, accept, sample, heat, q)
    assert _status_ok()


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("n", [33, 100, 1024])
def test_verify_large_trees(cuda_device, probs, n):
    rng = np.random.default_rng(n)
    for kind in ("chain", "star", "near"):
        trees = [_random_tree(rng, n, kind), _random_tree(rng, n // 2, kind)]
        logits, ids, accept, sample, heat, q = _verify_case(rng, trees, 37, probs)
        if kind == "chain":
            accept[:] = 0.0  # all the way down
        _check_verify(trees, logits, ids, accept, sample, heat, q)
    assert _status_ok()


def test_verify_values_that_are_no_numbers(cuda_device):
    nan, inf = np.nan, np.inf
    rows = np.array([[-inf, -inf, -inf, -inf], [nan, -inf, nan, nan], [nan, 1.0, -inf, 0.0], [inf, 1.0, inf, nan],
                     [-3.4e38, -3.4e38, 3.4e38, -inf], [1e-45, 0.0, -0.0, -1e-45]], np.float32)
    trees = [[-1]] * 6
    for u, heats in ((0.0, (1.0, 0.0, 1e-45, 3e38, inf)), (0.49, (1.0, 2.0)), (0.999, (1.0, 0.0))):
        for heat in heats:
            got = lq.verify_drafts(_f32(rows), _i32([0] * 6), _i32([-1] * 6), _plan([0] * 6, trees), _f32([0.0] * 6), _f32([u] * 6),
                                   _f32([heat] * 6))
            for s in range(6):
                # (3.4e38 apart, or 1e-45 with a heat of 1e-45: all or nothing, and e^-1 against 1)
                expect = od.verify(rows[s:s + 1], [0], [-1], [0.0], u, np.float32(min(heat, 3.4e38)))[1][-1]
                assert int(got.next[s]) == expect, (u, heat, s)
    # A draft behind such a row is not taken, and the walk ends there.
    logits = np.array([[0.0, 9.0, 0.0], [nan, nan, -inf], [0.0, 1.0, 2.0]], np.float32)
    got = lq.verify_drafts(_f32(logits), _i32([0, 1, 2]), _i32([-1, 0, 1]), _plan([0], [[-1, 0, 1]]), _f32([0.0] * 3), _f32([0.5]),
                           _f32([1.0]))
    assert got.path.tolist() == [[0, 1, -1]] and got.tokens.tolist() == [[1, -1, -1]]
    assert got.kept.tolist() == [2] and got.next.tolist() == [-1]
    # Draft probabilities that are none count as zero, uniform numbers outside [0, 1) as its ends.
    q = np.array([[nan, -1.0, 0.25]] * 3, np.float32)
    logits = np.log(np.array([[0.5, 0.25, 0.25]] * 3)).astype(np.float32)
    for sample, drawn in ((0.0, 0), (0.99, 1), (7.0, 1), (-3.0, 0), (nan, 0)):
        got = lq.verify_drafts(_f32(logits), _i32([0, 2, 2]), _i32([-1, 0, 0]), _plan([0], [[-1, 0, 0]]), _f32([0.0, 1.5, 2.0]),
                               _f32([sample]), _f32([1.0]), draft_probs=_f32(q))
        assert got.next.tolist() == [drawn] and got.kept.tolist() == [1]
    assert _status_ok()


@pytest.mark.parametrize("probs", [False, True])
def test_verify_where_nothing_is_left(cuda_device, probs):
    # A rejection that leaves no mass goes back to the target itself.
    logits = np.array([[0.0, -np.inf, -np.inf], [0.0] * 3, [0.0] * 3], np.float32)
    q = np.array([[1.0, 0.0, 0.0]] * 3, np.float32) if probs else None
    got = lq.verify_drafts(_f32(logits), _i32([0, 0, 0]), _i32([-1, 0, 0]), _plan([0], [[-1, 0, 0]]), _f32([0.0, 1.0, 0.5]),
                           _f32([0.5]), _f32([1.0]), draft_probs=None if q is None else _f32(q))
    assert got.path.tolist() == [[0, 2, -1]]
    got = lq.verify_drafts(_f32(logits), _i32([0, 0, 0]), _i32([-1, 0, 0]), _plan([0], [[-1, 0, 0]]), _f32([0.0, 1.0, 1.0]),
                           _f32([0.5]), _f32([1.0]), draft_probs=None if q is None else _f32(q))
    assert got.path.tolist() == [[0, -1, -1]] and got.next.tolist() == [0]


def test_verify_passes_over_ids_outside_the_vocabulary(cuda_device):
    logits = np.zeros((5, 8), np.float32)
    ids = [-9, 8, -1, 2**31 - 1, 3]
    got = lq.verify_drafts(_f32(logits), _i32(ids), _i32([-1, 0, 0, 0, 0]), _plan([0], [[-1, 0, 0, 0, 0]]), _f32([0.0] * 5),
                           _f32([0.5]), _f32([1.0]))
    assert got.path.tolist() == [[0, 4, -1, -1, -1]]
    assert _lib.load().leafq_device_status() == _lib.LEAFQ_ERR_INVALID
    got = lq.verify_drafts(_f32(logits[:1]), _i32([99]), _i32([-1]), _plan([0], [[-1]]), _f32([0.0]), _f32([0.5]), _f32([1.0]))
    assert got.kept.tolist() == [1] and _status_ok()  # row 0's own id is not looked at


def test_verify_follows_the_targets_distribution(cuda_device):
    # Drafts drawn from another distribution: what comes out first is drawn from the target's, whatever the drafts were.
    rng = np.random.default_rng(12)
    requests, vocab = 20000, 6
    p, q = rng.dirichlet(np.ones(vocab)), rng.dirichlet(np.ones(vocab))
    logits = np.tile(np.log(p).astype(np.float32), (4 * requests, 1))
    probs = np.tile(q.astype(np.float32), (4 * requests, 1))
    ids = rng.choice(vocab, 4 * requests, p=q)
    trees = [[-1, 0, 0, 0]] * requests
    got = lq.verify_drafts(_f32(logits), _i32(ids), _i32([-1, 0, 0, 0] * requests), _plan([0] * requests, trees),
                           _f32(rng.random(4 * requests)), _f32(rng.random(requests)), _f32(np.ones(requests)), draft_probs=_f32(probs))
    share = np.bincount(got.tokens[:, 0].cpu().numpy(), minlength=vocab) / requests
    assert np.all(np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / requests))  # five standard deviations
    kept = got.kept.cpu().numpy()
    assert 0.2 < (kept > 1).mean() < 1.0


def test_verify_streams_graphs_and_reuse(cuda_device):
    rng = np.random.default_rng(13)
    trees = [_random_tree(rng, int(n), "near") for n in rng.integers(1, 9, 40)]
    cases = [_verify_case(rng, trees, 999, True) for _ in range(2)]
    plan = _plan([0] * 40, trees)
    parents = _i32([p for t in trees for p in t])
    call = lambda c, **more: lq.verify_drafts(_f32(c[0]), _i32(c[1]), parents, plan, _f32(c[2]), _f32(c[3]), _f32(c[4]),  # noqa: E731
                                              draft_probs=_f32(c[5]), **more)
    expect = [[t.clone() for t in (v.path, v.tokens, v.kept, v.next)] for v in map(call, cases)]
    verdict = lq.Verdict(40, plan.max_tokens, "cuda")
    inputs = [[_f32(c[0]), _i32(c[1]), _f32(c[2]), _f32(c[3]), _f32(c[4]), _f32(c[5])] for c in cases]
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lq.verify_drafts(static[0], static[1], parents, plan, static[2], static[3], static[4], draft_probs=static[5], out=verdict)
    for _ in range(2):
        for values, e in zip(inputs, expect):
            for a, b in zip(static, values):
                a.copy_(b)
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip((verdict.path, verdict.tokens, verdict.kept, verdict.next), e))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        v = lq.verify_drafts(inputs[1][0], inputs[1][1], parents, plan, *inputs[1][2:5], draft_probs=inputs[1][5], out=verdict)
    side.synchronize()
    assert v is verdict and all(torch.equal(a, b) for a, b in zip((v.path, v.tokens, v.kept, v.next), expect[1]))
    assert _status_ok()


def test_calls_of_several_streams_at_once(cuda_device):
    # Each with its own workspace and outputs: both forms of the attention, causal tiles, and verification.
    rng = np.random.default_rng(61)
    batches = [_Trees(rng, [3000, 40], [70, 60], 16, 8, 8, 64, rotary=64), _Trees(rng, [900], [90], 64, 8, 8, 128),
               _Trees(rng, [100, 40], [5, 9], 16, 2, 4, 64, rotary=64)]
    trees = [_random_tree(rng, int(n), "near") for n in rng.integers(1, 9, 70)]
    logits, ids, accept, sample, heat, q = _verify_case(rng, trees, 4099, True)
    plan, parents = _plan([0] * 70, trees), _i32([p for t in trees for p in t])
    inputs = [_f32(logits), _i32(ids), parents, plan, _f32(accept), _f32(sample), _f32(heat), _f32(q)]
    rows = [torch.from_numpy(b.q).cuda() for b in batches]
    ropes = [_rope_cuda(b.rope) for b in batches]
    calls = [lambda w, b=b, x=x, r=r: lq.kv8_tree_attention(x, b.cache, b.plan, b.tree, b.scale, rope=r, workspace=w)
             for b, x, r in zip(batches, rows, ropes)]
    calls.append(lambda w: lq.kv8_attention(rows[0], batches[0].cache, batches[0].plan, batches[0].scale, rope=ropes[0], workspace=w))
    calls.append(lambda w: lq.verify_drafts(*inputs).path)
    expect = [call(lq.Kv8Workspace()) for call in calls]
    streams, workspaces = [torch.cuda.Stream() for _ in calls], [lq.Kv8Workspace() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(12):
        for out, call, stream, w in zip(got, calls, streams, workspaces):
            with torch.cuda.stream(stream):
                out.append(call(w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, e) for out, e in zip(got, expect) for o in out)
    assert _status_ok()


# ------------------------------------------------------------- a run of them
@pytest.mark.parametrize("page", [16, 64])
def test_a_step_of_drafts_end_to_end(cuda_device, page):
    """Plan, tree, append, tree attention, verify, compact, release: the cache afterwards is as near as its 8 bits
    to one that the accepted tokens alone were appended to, the pages are where the lengths say."""
    rng = np.random.default_rng(page)
    requests, kv, group, dim, layers, vocab = 6, 2, 4, 64, 3, 50
    pool, heads = 120, kv * group
    table, free, taken = _i32(np.full((requests, 20), -1)), _i32(rng.permutation(pool)), _i32([0])
    caches = [lq.Kv8Cache.empty(pool, kv, page, dim) for _ in range(layers)]
    stack = lq.Kv8Layers(caches)
    from test_gpu_kv8 import _rope
    rope_np = _rope(400, dim)
    rope = _rope_cuda(rope_np)
    length = _i32(np.zeros(requests))
    truth = [[[] for _ in range(requests)] for _ in range(layers)]  # the accepted tokens' (k, v), k rotated
    largest = np.zeros((layers, 2, kv))  # scale that any page has had
    for step in range(6):
        sizes = rng.integers(30, 60, requests) if step == 0 else rng.integers(0, 20, requests)
        trees = [_random_tree(rng, int(n), "chain" if step == 0 else "near") if n else [] for n in sizes]
        tokens = int(sizes.sum())
        before = length.tolist()
        plan = lq.kv8_plan(length, _i32(sizes), table, free, taken, page, tokens, max_tokens=int(sizes.max()))
        parents = _i32([p for t in trees for p in t])
        tree = lq.kv8_tree(parents, plan)
        logits, ids, accept, sample, heat, q = _verify_case(rng, trees, vocab, True)
        if step == 0:
            accept[:] = 0.0  # prompts stand
        verdict = lq.verify_drafts(_f32(logits), _i32(ids), parents, plan, _f32(accept), _f32(sample), _f32(heat), draft_probs=_f32(q))
        kept, path = verdict.kept.tolist(), verdict.path.tolist()
        offsets = plan.token_offsets.tolist()
        positions = tree.positions.cpu().numpy()
        for i, cache in enumerate(caches):
            qkv = rng.standard_normal((tokens, (heads + 2 * kv) * dim)).astype(np.float32)
            x = torch.from_numpy(qkv).cuda()
            k, v = x[:, heads * dim:(heads + kv) * dim], x[:, (heads + kv) * dim:]
            lq.kv8_append(k, v, cache, plan.slots, tree.positions, rope=rope)
            out = lq.kv8_tree_attention(x[:, :heads * dim], cache, plan, tree, dim ** -0.5, rope=rope)
            # against the cache's values and the tree
            k_all, v_all = (t.cpu().numpy().astype(np.float64) for t in (cache.k, cache.v))
            k_s, v_s = (t.cpu().numpy().astype(np.float64) for t in (cache.k_scale, cache.v_scale))
            turned = ok.rotate(qkv[:, :heads * dim].reshape(tokens, heads, dim), positions, rope_np)
            rows = table.cpu().numpy()
            used = [p for s in range(requests) for p in rows[s, :ok.pages_of(before[s] + int(sizes[s]), page)].tolist()]
            largest[i] = np.maximum(largest[i], [k_s[used].max(axis=0), v_s[used].max(axis=0)])
            for s in range(requests):
                n, c = int(sizes[s]), before[s]
                held = rows[s, :ok.pages_of(c + n, page)]
                seen = np.zeros((n, held.size * page), dtype=bool)
                for t, above in enumerate(ok.tree(trees[s], c)[1]):
                    seen[t, :c] = True
                    seen[t, [c + a for a in above]] = True
                for h in range(kv):
                    kk = (k_all[held, h] * k_s[held, h][:, None, None]).reshape(-1, dim)
                    vv = (v_all[held, h] * v_s[held, h][:, None, None]).reshape(-1, dim)
                    want, _ = ok.tree_attention(turned[offsets[s]:offsets[s + 1], h * group:(h + 1) * group], seen, kk, vv, dim ** -0.5)
                    got = out[offsets[s]:offsets[s + 1]].reshape(n, heads, dim)[:, h * group:(h + 1) * group].cpu().numpy()
                    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)
            k_turned = ok.rotate(qkv[:, heads * dim:(heads + kv) * dim].reshape(tokens, kv, dim), positions, rope_np)
            for s in range(requests):
                for t in path[s][:kept[s]]:
                    truth[i][s].append((k_turned[offsets[s] + t], qkv[offsets[s] + t, (heads + kv) * dim:].reshape(kv, dim)))
        lq.kv8_compact(stack, plan, verdict.path, verdict.kept)
        left = lq.kv8_release(plan, verdict.kept, free, plan.taken)
        length.copy_(left.lengths)
        taken.copy_(left.taken)
        assert length.tolist() == [b + k for b, k in zip(before, kept)]
        rows = table.cpu().numpy()
        held = [p for s in range(requests) for p in rows[s, :ok.pages_of(int(length[s]), page)].tolist()]
        assert sorted(held + free.tolist()[int(taken):]) == list(range(pool))
        # Every value is within the roundings that its row went through, half a scale each (of the largest that there
        # was: a compaction's are no larger than those that rows come from): the row's append, its move, and in every
        # step the page's scale may grow twice.
        for i, cache in enumerate(caches):
            for s in range(requests):
                n = int(length[s])
                pages = rows[s, :ok.pages_of(n, page)]
                for side, codes, scales in ((0, cache.k, cache.k_scale), (1, cache.v, cache.v_scale)):
                    c, sc = (t[pages.tolist()].cpu().numpy().astype(np.float64) for t in (codes, scales))
                    values = (c * sc[:, :, None, None]).transpose(0, 2, 1, 3).reshape(-1, kv, dim)[:n]
                    want = np.array([pair[side] for pair in truth[i][s]])
                    assert values.shape == want.shape
                    assert np.all(np.abs(values - want) <= 0.5 * (2 + 2 * (step + 1)) * largest[i, side][:, None] * (1 + 1e-5))
    assert _status_ok()
