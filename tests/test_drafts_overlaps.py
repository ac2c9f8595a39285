"""Calls that check drafted tokens refuse outputs that share memory with what others of their blocks still read,
on the host, before touching a device."""
import ctypes

import pytest
import torch

import leaf_b200 as lq
from leaf_b200 import _lib

# Of the verification: 3 requests, 8 rows of 100 logits (strides of 120 and 110 floats), trees of up to 4 rows.
REQUESTS, TOKENS, MOST, VOCAB = 3, 8, 4, 100
INPUTS = dict(logits=(7 * 120 + VOCAB, 1 << 16), draft_probs=(7 * 110 + VOCAB, 2 << 16), ids=(TOKENS, 3 << 16),
              parents=(TOKENS, 4 << 16), token_offsets=(REQUESTS + 1, 5 << 16), accept=(TOKENS, 6 << 16), sample=(REQUESTS, 7 << 16),
              temperature=(REQUESTS, 8 << 16))
OUTPUTS = dict(path=(REQUESTS * MOST, 9 << 16), tokens=(REQUESTS * MOST, 10 << 16), kept=(REQUESTS, 11 << 16), next=(REQUESTS, 12 << 16))


def _verify(**moved):
    at = {name: ctypes.c_void_p(moved.get(name, where)) for name, (_, where) in (INPUTS | OUTPUTS).items()}
    return _lib.load().leafq_verify_drafts(None, at["logits"], 120, VOCAB, at["ids"], at["parents"], at["token_offsets"], REQUESTS,
                                           TOKENS, MOST, at["accept"], at["sample"], at["temperature"], at["draft_probs"], 110,
                                           at["path"], at["tokens"], at["kept"], at["next"], 0)


@pytest.mark.parametrize("output", list(OUTPUTS))
@pytest.mark.parametrize("other", list(INPUTS | OUTPUTS))
def test_verify_refuses_outputs_over_what_it_reads(output, other):
    if output == other:
        return
    count, where = (INPUTS | OUTPUTS)[other]
    own = OUTPUTS[output][0]
    for at in (where, where + 4 * (count - 1), where - 4 * (own - 1)):  # the same place; its last value; the output's last its first
        assert _verify(**{output: at}) == _lib.LEAFQ_ERR_INVALID
        assert b"overlap" in _lib.load().leafq_last_error()


def test_verify_without_probabilities_looks_at_the_others():
    offsets = INPUTS["token_offsets"][1]
    assert _verify(draft_probs=None, kept=offsets) == _lib.LEAFQ_ERR_INVALID and b"overlap" in _lib.load().leafq_last_error()
    assert _verify(draft_probs=None, tokens=INPUTS["ids"][1]) == _lib.LEAFQ_ERR_INVALID


# Of the compaction: 8 pages of 2 heads, 64 tokens and 64 values: 65,536 bytes of codes, 64 of scales a pool.
def _compact(*pools):
    caches = (_lib.Kv8CacheDesc * len(pools))(*(_lib.Kv8CacheDesc(*p, 8, 64, 2, 64) for p in pools))
    step = _lib.Kv8StepDesc(context=256, lengths=256, token_offsets=256, page_offsets=256, table=256, max_pages=4, tokens=3,
                            max_tokens=1, requests=3)
    where = ctypes.c_void_p(256)
    return _lib.load().leafq_kv8_compact(None, caches, len(pools), ctypes.byref(step), where, 4, where, 0)


def _apart(i):
    return [(i + 1) << 20, ((i + 1) << 20) + 65536, ((i + 1) << 20) + 131072, ((i + 1) << 20) + 131136]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("layers", [1, 2, 40])
def test_compact_refuses_pools_that_share_memory(which, layers):
    caches = [_apart(i) for i in range(layers)]
    last = caches[-1]
    for victim in range(4):
        if layers == 1 and victim == which:
            continue
        begin, size = caches[0][victim], 65536 if victim < 2 else 64
        for at in (begin, begin + size - 16):
            moved = [*caches[:-1], [*last[:which], at, *last[which + 1:]]]
            assert _compact(*moved) == _lib.LEAFQ_ERR_INVALID
            assert b"memory of another" in _lib.load().leafq_last_error()


def test_layers_refuse_caches_that_share_memory():
    def cache(pools):
        c = lq.Kv8Cache.__new__(lq.Kv8Cache)
        c.k, c.v, c.k_scale, c.v_scale = pools
        c.index, c.pages, c.page, c.kv_heads, c.dim = 0, 2, 16, 1, 32
        c.desc = _lib.Kv8CacheDesc(*(t.data_ptr() for t in pools), 2, 16, 1, 32)
        return c

    pool = torch.zeros(9000, dtype=torch.int8)
    scales = torch.zeros(64)
    def pools(at, scale_at):
        return [pool[at:at + 1024].view(2, 1, 16, 32), pool[at + 1024:at + 2048].view(2, 1, 16, 32),
                scales[scale_at:scale_at + 2].view(2, 1), scales[scale_at + 2:scale_at + 4].view(2, 1)]

    assert len(lq.Kv8Layers([cache(pools(0, 0)), cache(pools(2048, 4)), cache(pools(4096, 8))]).caches) == 3
    for second in (pools(1024, 4), pools(2032, 4), pools(2048, 3), pools(0, 0)):
        with pytest.raises(lq.LeafError, match="memory of another"):
            lq.Kv8Layers([cache(pools(0, 0)), cache(second)])
    # A page of another pool, whose first one it is not.
    with pytest.raises(lq.LeafError, match="memory of another"):
        lq.Kv8Layers([cache(pools(4096, 8)), cache(pools(4096 + 512, 20))])
