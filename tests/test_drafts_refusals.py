"""The entry points that check drafted tokens reject invalid arguments on the host, before touching a device."""
import ctypes

import pytest
import torch

import leaf_b200 as lq
from leaf_b200 import _lib

P = ctypes.c_void_p(256)
Q = ctypes.c_void_p(1 << 20)
R = ctypes.c_void_p(1 << 21)
ODD = ctypes.c_void_p(264)


def _cache(**change):
    fields = dict(k_codes=256, v_codes=256, k_scales=256, v_scales=256, pages=8, page=64, kv_heads=2, dim=64)
    fields.update(change)
    return _lib.Kv8CacheDesc(**fields)


def _step(**change):
    fields = dict(context=256, lengths=256, token_offsets=256, page_offsets=256, table=256, max_pages=4, tokens=3,
                  max_tokens=1, requests=3)
    fields.update(change)
    return _lib.Kv8StepDesc(**fields)


def _tree(step=None, parents=P, positions=Q, masks=R, words=1):
    step = _step() if step is None else step
    return _lib.load().leafq_kv8_tree(None, parents, ctypes.byref(step) if step else None, positions, masks, words, 0)


@pytest.mark.parametrize("change", [dict(step=False), dict(step=_step(tokens=-1)), dict(step=_step(tokens=2**31)),
                                    dict(step=_step(requests=-1)), dict(step=_step(max_tokens=-1)), dict(words=0),
                                    dict(words=33), dict(step=_step(max_tokens=33)), dict(parents=None), dict(positions=None),
                                    dict(masks=None), dict(step=_step(token_offsets=None)), dict(step=_step(context=None)),
                                    dict(positions=P), dict(masks=P), dict(masks=Q), dict(positions=ctypes.c_void_p(256 + 8)),
                                    dict(masks=ctypes.c_void_p((1 << 20) + 8))])
def test_tree_rejects(change):
    assert _tree(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def test_trees_of_too_many_rows():
    assert _tree(step=_step(max_tokens=1025), words=32) == _lib.LEAFQ_ERR_UNSUPPORTED
    assert _verify(most=1025) == _lib.LEAFQ_ERR_UNSUPPORTED
    assert _verify(vocab=2**20 + 1, stride=2**21, probs_stride=2**21) == _lib.LEAFQ_ERR_UNSUPPORTED


def _attend(cache=None, step=None, q=P, stride=256, heads=4, rotary=0, cos=None, sin=None, rows=0, positions=P, masks=P, words=1,
            scale=0.125, out=P, workspace=P, nbytes=1 << 40):
    cache, step = _cache() if cache is None else cache, _step() if step is None else step
    return _lib.load().leafq_kv8_tree_attention(None, q, stride, heads, rotary, cos, sin, rows, ctypes.byref(cache),
                                                ctypes.byref(step) if step else None, positions, masks, words, scale, out, workspace,
                                                nbytes, 0)


@pytest.mark.parametrize("change", [dict(cache=_cache(page=8)), dict(step=False), dict(step=_step(tokens=-1)),
                                    dict(step=_step(requests=-1)), dict(step=_step(max_pages=2**31 // 64)),
                                    dict(step=_step(context=None)), dict(step=_step(table=None)), dict(heads=5),
                                    dict(scale=float("nan")), dict(q=None), dict(out=ODD), dict(stride=255), dict(positions=None),
                                    dict(masks=None), dict(words=0), dict(words=33), dict(step=_step(max_tokens=33)),
                                    dict(rotary=64), dict(nbytes=0), dict(workspace=None)])
def test_tree_attention_rejects(change):
    assert _attend(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def _compact(caches=None, layers=None, step=None, path=P, width=4, kept=P):
    caches = [_cache(), _cache()] if caches is None else caches
    array = (_lib.Kv8CacheDesc * max(1, len(caches)))(*caches)
    step = _step() if step is None else step
    return _lib.load().leafq_kv8_compact(None, array, len(caches) if layers is None else layers, ctypes.byref(step) if step else None,
                                         path, width, kept, 0)


@pytest.mark.parametrize("change", [dict(layers=-1), dict(step=False), dict(step=_step(requests=-1)), dict(width=-1),
                                    dict(width=1025), dict(path=None), dict(kept=None), dict(step=_step(context=None)),
                                    dict(step=_step(lengths=None)), dict(step=_step(table=None)),
                                    dict(caches=[_cache(), _cache(page=32)]), dict(caches=[_cache(), _cache(kv_heads=1)]),
                                    dict(caches=[_cache(), _cache(dim=128)]), dict(caches=[_cache(), _cache(pages=9)]),
                                    dict(caches=[_cache(k_codes=None)]), dict(caches=[_cache(), _cache(v_codes=264)])])
def test_compact_rejects(change):
    assert _compact(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def _release(step=None, kept=P, page=64, free=Q, count=8, taken=P, lengths=R, after=ODD):
    step = _step(context=512, lengths=1024, table=2048) if step is None else step
    return _lib.load().leafq_kv8_release(None, ctypes.byref(step) if step else None, kept, page, free, count, taken, lengths, after, 0)


@pytest.mark.parametrize("change", [dict(step=False), dict(step=_step(requests=-1)), dict(page=0), dict(page=48), dict(count=-1),
                                    dict(count=2**31), dict(step=_step(max_pages=2**31 // 64)), dict(kept=None), dict(free=None),
                                    dict(taken=None), dict(lengths=None), dict(after=None), dict(step=_step(lengths=None)),
                                    dict(after=P), dict(lengths=ctypes.c_void_p(1024)), dict(free=ctypes.c_void_p(2048 + 40)),
                                    dict(lengths=Q), dict(after=ctypes.c_void_p((1 << 21) + 8)), dict(lengths=ctypes.c_void_p(512 + 8))])
def test_release_rejects(change):
    assert _release(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def _verify(logits=P, stride=100, vocab=100, ids=P, parents=P, offsets=P, requests=2, tokens=4, most=2, accept=P, sample=P, heat=P,
            probs=P, probs_stride=100, path=P, out=P, kept=P, nxt=P):
    return _lib.load().leafq_verify_drafts(None, logits, stride, vocab, ids, parents, offsets, requests, tokens, most, accept, sample,
                                           heat, probs, probs_stride, path, out, kept, nxt, 0)


@pytest.mark.parametrize("change", [dict(vocab=0), dict(vocab=-5), dict(requests=-1), dict(requests=2**31 // 8), dict(tokens=-1), dict(tokens=2**31), dict(most=-1),
                                    dict(stride=99), dict(probs_stride=99), dict(logits=None), dict(ids=None), dict(parents=None),
                                    dict(offsets=None), dict(accept=None), dict(sample=None), dict(heat=None), dict(path=None),
                                    dict(out=None), dict(kept=None), dict(nxt=None)])
def test_verify_rejects(change):
    assert _verify(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def test_unsupported_head_sizes():
    for dim in (16, 48, 80, 160, 256):
        assert _attend(cache=_cache(dim=dim), stride=4096) == _lib.LEAFQ_ERR_UNSUPPORTED
        assert _compact(caches=[_cache(dim=dim)]) == _lib.LEAFQ_ERR_UNSUPPORTED


def test_empty_calls_are_no_ops():
    assert _tree(step=_step(tokens=0, max_tokens=0), parents=None, positions=None, masks=None) == 0
    assert _attend(step=_step(tokens=0), q=None, out=None, positions=None, masks=None) == 0
    assert _attend(step=_step(requests=0), q=None, out=None) == 0
    assert _compact(layers=0) == 0
    assert _compact(step=_step(requests=0), path=None, kept=None) == 0
    assert _compact(width=0, path=None) == 0
    assert _verify(requests=0, logits=None, path=None) == 0


def test_python_refuses_what_it_cannot_pass_on():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(lq.LeafError, match="int32 CUDA"):
        lq.Kv8Tree(i(4), i(4, 1))
    with pytest.raises(lq.LeafError, match="there must be a layer"):
        lq.Kv8Layers([])
    def cache(pools):
        c = lq.Kv8Cache.__new__(lq.Kv8Cache)
        c.k, c.v, c.k_scale, c.v_scale = pools
        c.index, c.pages, c.page, c.kv_heads, c.dim = 0, 2, 16, 1, 32
        c.desc = lq._lib.Kv8CacheDesc(*(t.data_ptr() for t in pools), 2, 16, 1, 32)
        return c
    apart = [[torch.zeros(4) for _ in range(4)] for _ in range(2)]
    assert len(lq.Kv8Layers([cache(p) for p in apart]).caches) == 2
    for twice in ([apart[0], apart[0]], [apart[0], [*apart[1][:3], apart[0][0]]]):  # both would be moved at once
        with pytest.raises(lq.LeafError, match="a cache is there twice"):
            lq.Kv8Layers([cache(p) for p in twice])
    with pytest.raises(lq.LeafError, match="tree is missing"):
        lq.kv8_tree_attention(torch.zeros(1, 64), None, None, None, 0.125)
    with pytest.raises(lq.LeafError, match="int32 CUDA"):
        lq.Kv8Released(i(2), i(1))


class _Device:
    """Handles that look like those of tensors on a GPU, so that the checks in front of a launch run here."""

    def __init__(self, monkeypatch, index=0):
        from leaf_b200 import drafts, kv8
        for module in (drafts, kv8):
            monkeypatch.setattr(module, "_current_device", lambda: index)
            monkeypatch.setattr(module, "_raw_stream", lambda i: None)
        monkeypatch.setattr(kv8, "_check_i32", self.check)
        monkeypatch.setattr(drafts, "_check_i32", self.check)
        self.index = index

    @staticmethod
    def check(t, name, numel=None, index=None):
        if numel is not None and t.numel() != numel:
            raise lq.LeafError(1, f"{name} must hold {numel} values")

    def plan(self, requests=2, tokens=5, most=4, page=16):
        plan = lq.Kv8Plan.__new__(lq.Kv8Plan)
        plan.requests, plan.tokens, plan.max_tokens, plan.index, plan.page, plan.device = requests, tokens, most, self.index, page, "cpu"
        return plan


def test_python_refuses_other_sizes(monkeypatch):
    from leaf_b200 import kv8
    device = _Device(monkeypatch)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    plan = device.plan()
    with pytest.raises(lq.LeafError, match="parents must hold 5"):
        lq.kv8_tree(i(4), plan)
    with pytest.raises(lq.LeafError, match="at most 1024 rows"):
        lq.kv8_tree(i(5), device.plan(most=1025))
    tree = kv8.Kv8Tree(i(4), i(4, 1))
    tree.index = 0
    with pytest.raises(lq.LeafError, match="tree is of other rows"):
        lq.kv8_tree(i(5), plan, out=tree)
    with pytest.raises(lq.LeafError, match="page size is not known"):
        lq.kv8_release(device.plan(page=None), i(2), i(8), i(1))
    left = kv8.Kv8Released(i(3), i(1))
    left.index = 0
    with pytest.raises(lq.LeafError, match="other requests"):
        lq.kv8_release(plan, i(2), i(8), i(1), out=left)
    layers = kv8.Kv8Layers.__new__(kv8.Kv8Layers)
    layers.index, layers.page = 0, 32
    with pytest.raises(lq.LeafError, match="pages of 16 tokens, the caches of 32"):
        lq.kv8_compact(layers, plan, i(2, 4), i(2))
    layers.page = 16
    with pytest.raises(lq.LeafError, match="path must be"):
        lq.kv8_compact(layers, plan, i(3, 4), i(2))
    layers.index = 1
    monkeypatch.setattr(kv8, "_current_device", lambda: 1)
    with pytest.raises(lq.LeafError, match="another device"):
        lq.kv8_compact(layers, plan, i(2, 4), i(2))
    f = torch.zeros
    with pytest.raises(lq.LeafError, match=r"logits must be float32"):
        lq.verify_drafts(f(5, 9, dtype=torch.float16), i(5), i(5), plan, f(5), f(2), f(2))
