"""The decoder over the paged INT8 cache.

* Every append and attention of a run is held, with the decoder's own inputs,
  to the definitions in oracle/kv8.py, at the tolerances of test_gpu_kv8.py.
* The first layer's attention of a prompt is held to unquantised attention in
  64-bit floats.  Keys and values of a page are rounded once, by half a step at
  most (dk, dv), so scores move by at most e = scale * |q|_1 * dk and weights by
  a factor within exp(2 e): |difference| <= (exp(2 e) - 1) * max |v| + dv, plus
  1e-5 of max |v| for the float32 sums (rounding of the kind above is 1e-6).
* The step's graph, a second run and steps without the graph give equal bits.
"""
import json

import numpy as np
import pytest
import torch

import leaf_b200.decoder as module
from conftest import GOLDEN
from leaf_b200 import LeafError
from leaf_b200.decoder import Decoder
import decoder_fixture as fx  # tests/golden
from oracle import kv8 as ok
from oracle.fixture import LlamaShape

U = 2.0 ** -24


def _artifact(tmp_path, name="tiny_w8", shape=fx.TINY):
    meta = json.loads((GOLDEN / f"decoder_{name}.json").read_text())
    path = tmp_path / f"{name}.leaf"
    tensors = fx.llama_tensors(shape, meta["weight_seed"], meta["norm_noise"])
    extras = ()
    if name == "tiny_smooth":
        tensors, extras = fx.smooth_variant(shape, tensors, meta["weight_seed"] + 1)
    fx.write_artifact(path, shape, tensors, meta["bits"], meta["group"], extras=extras)
    return path


class _Watch:
    """Holds each kv8 call of a decoder to its definition."""

    def __init__(self, monkeypatch, dec):
        self.dec, self.calls, self.first = dec, 0, None
        self.append, self.attention = module.kv8_append, module.kv8_attention
        monkeypatch.setattr(module, "kv8_append", self.on_append)
        monkeypatch.setattr(module, "kv8_attention", self.on_attention)

    @staticmethod
    def host(t):
        return t.detach().cpu().numpy().copy()

    def on_append(self, k, v, cache, slots, positions, rope):
        before = [self.host(t) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        self.append(k, v, cache, slots, positions, rope=rope)
        tables = tuple(self.host(t) for t in rope)
        heads, dim = cache.kv_heads, cache.dim
        live = self.host(slots)
        n = int((live >= 0).sum())
        assert np.all(live[:n] >= 0)
        for i, (x, got, got_scale) in enumerate(((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale))):
            x = self.host(x).reshape(-1, heads, dim)[:n]
            if i == 0:
                x = ok.rotate(x, self.host(positions)[:n], tables)
            scales = np.where(np.isfinite(before[2 + i]), before[2 + i], 0.0)  # pages not yet written
            expect, expect_scale, real = ok.append(x, live[:n], before[i], scales)
            got, got_scale = self.host(got), self.host(got_scale)
            held = np.unique(live[:n] // cache.page)
            assert np.all(np.abs(got_scale[held] - expect_scale[held]) <= 8 * U * expect_scale[held])
            differ = (got != expect)[held]
            tie = (np.abs(np.abs(real - np.floor(real)) - 0.5) < 127 * 16 * U)[held]
            assert not np.any(differ & ~tie)
        self.calls += 1

    def on_attention(self, q, cache, plan, scale, rope, out, workspace):
        self.attention(q, cache, plan, scale, rope=rope, out=out, workspace=workspace)
        heads, kv, dim, page = q.shape[1] // cache.dim, cache.kv_heads, cache.dim, cache.page
        group, tables = heads // kv, tuple(self.host(t) for t in rope)
        offsets, context, lengths, table = (self.host(t) for t in (plan.token_offsets, plan.context, plan.lengths, plan.table))
        queries, got = self.host(q), self.host(out)
        codes = [self.host(t).astype(np.float64) for t in (cache.k, cache.v)]
        scales = [self.host(t).astype(np.float64) for t in (cache.k_scale, cache.v_scale)]
        for s in range(plan.requests):
            rows = slice(offsets[s], offsets[s + 1])
            positions = context[s] + np.arange(offsets[s + 1] - offsets[s])
            x = ok.rotate(queries[rows].reshape(-1, heads, dim), positions, tables)
            held, n = table[s, :ok.pages_of(lengths[s], page)], lengths[s]
            for h in range(kv):
                k, v = ((codes[i][held, h] * scales[i][held, h][:, None, None]).reshape(-1, dim)[:n] for i in range(2))
                expect, reach = ok.attention(x[:, h * group:(h + 1) * group], positions + 1, k, v, scale)
                part = got[rows].reshape(-1, heads, dim)[:, h * group:(h + 1) * group]
                bound = np.abs(v).max() * (2 * (dim + 16) * reach + 64) * U
                assert np.all(np.abs(part - expect) <= bound[..., None])
        if self.first is None:
            self.first = (queries, got)
        self.calls += 1


def _prompt(rng, shape, n):
    return [int(i) for i in rng.integers(0, shape.vocab, n)]


@pytest.mark.gpu
@pytest.mark.parametrize("name,page,bits", [("tiny_w8", 16, 8), ("tiny_w4", 32, 8), ("tiny_smooth", 64, 32)])
def test_every_call_of_a_ragged_batch(cuda_device, tmp_path, monkeypatch, name, page, bits):
    rng = np.random.default_rng(page)
    dec = Decoder(_artifact(tmp_path, name), activation_bits=bits, sequences=3, cache="int8", page=page)
    watch = _Watch(monkeypatch, dec)
    lengths = [5, 70, 33]
    dec.forward_batch([_prompt(rng, fx.TINY, n) for n in lengths])
    for new in ([1, 1, 1], [1, 1, 1], [4, 1, 9]):
        dec.forward_batch([_prompt(rng, fx.TINY, n) for n in new])
        lengths = [a + b for a, b in zip(lengths, new)]
        assert dec.position.tolist() == lengths
    assert watch.calls == 4 * 2 * fx.TINY.layers
    assert int(dec.taken) == sum(ok.pages_of(n, page) for n in lengths)
    assert dec.device_status() == 0
    dec.reset()  # the pages are free again, whatever they hold
    dec.forward_batch([_prompt(rng, fx.TINY, n) for n in (40, 3, 18)])
    assert dec.position.tolist() == [40, 3, 18]


@pytest.mark.gpu
def test_first_layer_is_near_unquantised_attention(cuda_device, tmp_path, monkeypatch):
    shape, n = fx.TINY, 90
    dec = Decoder(_artifact(tmp_path), cache="int8", page=64)
    watch = _Watch(monkeypatch, dec)
    dec.forward(_prompt(np.random.default_rng(1), shape, n))
    queries, got = watch.first
    # What entered the first layer's cache, again: the prompt's projections.
    dec2 = Decoder(_artifact(tmp_path), cache="int8", page=64)
    rows = []
    monkeypatch.setattr(module, "kv8_append", lambda k, v, *a, **kw: (rows.append((watch.host(k), watch.host(v))),
                                                                      watch.append(k, v, *a, **kw)))
    monkeypatch.setattr(module, "kv8_attention", watch.attention)
    dec2.forward(_prompt(np.random.default_rng(1), shape, n))
    dim, kv, group = shape.head_dim, shape.kv_heads, shape.heads // shape.kv_heads
    tables = tuple(watch.host(t) for t in (dec.cos, dec.sin))
    at = np.arange(n)
    q = ok.rotate(queries.reshape(n, shape.heads, dim), at, tables)
    k = ok.rotate(rows[0][0].reshape(n, kv, dim), at, tables)
    v = rows[0][1].reshape(n, kv, dim).astype(np.float64)
    scale = dim ** -0.5
    for h in range(kv):
        x = q[:, h * group:(h + 1) * group]
        expect, _ = ok.attention(x, at + 1, k[:, h], v[:, h], scale)
        dk, dv = np.abs(k[:, h]).max() / 254, np.abs(v[:, h]).max() / 254
        e = scale * np.abs(x).sum(axis=2) * dk
        bound = (np.exp(2 * e) - 1) * np.abs(v[:, h]).max() + dv + 1e-5 * np.abs(v[:, h]).max()
        part = got.reshape(n, shape.heads, dim)[:, h * group:(h + 1) * group]
        assert np.all(np.abs(part - expect) <= bound[..., None])


@pytest.mark.gpu
@pytest.mark.parametrize("sequences,page", [(1, 16), (4, 64)])
def test_graph_steps_and_repeats_are_equal(cuda_device, tmp_path, sequences, page):
    path, rng = _artifact(tmp_path), np.random.default_rng(7)
    prompts = [_prompt(rng, fx.TINY, 20 + 13 * s) for s in range(sequences)]
    steps = 40
    dec = Decoder(path, sequences=sequences, cache="int8", page=page)
    first = dec.generate_batch(prompts, steps)
    assert dec.position.tolist() == [len(p) + steps - 1 for p in prompts]
    logits = dec._bufs(1)["logits"].clone()
    dec.reset()
    assert dec.generate_batch(prompts, steps) == first
    assert torch.equal(dec._bufs(1)["logits"], logits)
    plain = Decoder(path, sequences=sequences, cache="int8", page=page)
    out = plain.forward_batch(prompts)
    for i in range(steps - 1):
        assert out.argmax(dim=1).tolist() == [f[i] for f in first]
        out = plain.forward_batch([[f[i]] for f in first])
    assert torch.equal(out, logits)
    if sequences == 1:
        dec.reset()
        assert dec.generate(prompts[0], steps) == first[0]
    assert dec.device_status() == 0 and plain.device_status() == 0


@pytest.mark.gpu
def test_capture_in_the_middle_keeps_the_pages(cuda_device, tmp_path):
    path, rng = _artifact(tmp_path), np.random.default_rng(8)
    prompt = _prompt(rng, fx.TINY, 31)
    early, late = (Decoder(path, cache="int8", page=16) for _ in range(2))
    early.capture_decode()
    outs = []
    for dec in (early, late):
        dec.forward(prompt)
        if dec is late:
            dec.capture_decode()
        assert int(dec.taken) == 2 and dec.position.tolist() == [31]
        outs.append(dec.generate(prompt[:5], 12))
    assert outs[0] == outs[1]


@pytest.mark.gpu
def test_tinyllama_heads_follow_the_fp32_cache(cuda_device, tmp_path):
    """64-wide heads, 8 queries a key: the tokens of a prompt's own logits
    stay what the fp32 cache gives where its margin is clear of 8-bit noise."""
    shape = LlamaShape(hidden=512, intermediate=512, heads=8, kv_heads=1, layers=2, vocab=512, max_positions=700)
    path = tmp_path / "heads64.leaf"
    fx.write_artifact(path, shape, fx.llama_tensors(shape, 3, 0.1), 8, 0)
    prompt = _prompt(np.random.default_rng(2), shape, 600)  # long enough for the tensor-core tiles
    a = Decoder(path, activation_bits=32).forward(prompt)[0].double()
    b = Decoder(path, activation_bits=32, cache="int8").forward(prompt)[0].double()
    # Codes are within 1/254 of their page's largest: attention within a few
    # hundredths of its own size, and the logits, which the residual stream
    # carries as well, no worse.
    assert float((a - b).norm() / a.norm()) < 0.05


@pytest.mark.gpu
def test_refusals(cuda_device, tmp_path):
    path = _artifact(tmp_path)
    with pytest.raises(LeafError):
        Decoder(path, cache="int4")
    with pytest.raises(LeafError):
        Decoder(path, cache="int8", page=48)
    dec = Decoder(path, sequences=2)
    with pytest.raises(LeafError):
        dec.forward_batch([[1, 2], [3]])  # unlike lengths need the INT8 cache
    dec = Decoder(path, sequences=2, cache="int8")
    for prompts in ([[1, 2], []], [[1]], [[1], [fx.TINY.vocab]], [[1], [1] * (fx.TINY.max_positions + 1)]):
        with pytest.raises(LeafError):
            dec.forward_batch(prompts)
    assert dec.position.tolist() == [0, 0]
    one = Decoder(path, cache="int8")
    assert not one.fused_supported()
    with pytest.raises(LeafError):
        one.generate_fused([1, 2, 3], 2)


@pytest.mark.gpu
def test_unlike_steps_fill_the_capacity(cuda_device, tmp_path):
    # Two steps of 1 and 100 tokens the other way round hold 101 each, and leave room for the rest.
    rng = np.random.default_rng(9)
    dec = Decoder(_artifact(tmp_path), sequences=2, capacity=128, cache="int8", page=16)
    for lengths in ((1, 100), (100, 1)):
        dec.forward_batch([_prompt(rng, fx.TINY, n) for n in lengths])
    assert dec.position.tolist() == [101, 101] and dec.length == 101
    dec.forward_batch([_prompt(rng, fx.TINY, n) for n in (7, 2)])
    with pytest.raises(LeafError):
        dec.forward_batch([_prompt(rng, fx.TINY, n) for n in (21, 1)])  # the longer one is at 108
    with pytest.raises(LeafError):
        dec.generate_batch([_prompt(rng, fx.TINY, n) for n in (1, 18)], 21)
    tokens = dec.generate_batch([_prompt(rng, fx.TINY, n) for n in (1, 18)], 8)
    assert [len(t) for t in tokens] == [8, 8] and dec.position.tolist() == [116, 128] and dec.length == 128
    with pytest.raises(LeafError):
        dec.forward_batch([[1], [1]])
    assert dec.device_status() == 0
    dec.reset()
    dec.forward_batch([_prompt(rng, fx.TINY, n) for n in (128, 1)])
    assert dec.length == 128
