"""The paged INT8 cache's entry points reject invalid arguments on the host,
before touching a device."""
import ctypes
import types
import weakref

import pytest
import torch

import leaf_b200 as lq
from leaf_b200 import _lib
from leaf_b200 import kv8

P = ctypes.c_void_p(256)
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


def _plan(context=P, new=P, requests=3, table=P, max_pages=4, free=P, free_count=8, taken=P, page=64, tokens=3, lengths=P,
          token_offsets=P, page_offsets=P, positions=P, slots=P, after=P):
    return _lib.load().leafq_kv8_plan(None, context, new, requests, table, max_pages, free, free_count, taken, page, tokens,
                                      lengths, token_offsets, page_offsets, positions, slots, after, 0)


@pytest.mark.parametrize("change", [dict(requests=-1), dict(max_pages=-1), dict(free_count=-1), dict(tokens=-1),
                                    dict(page=0), dict(page=48), dict(page=256), dict(max_pages=2**31 // 64),
                                    dict(tokens=2**31), dict(context=None), dict(new=None), dict(table=None),
                                    dict(free=None), dict(taken=None), dict(lengths=None), dict(token_offsets=None),
                                    dict(page_offsets=None), dict(positions=None), dict(slots=None), dict(after=None),
                                    dict(positions=ODD), dict(slots=ODD)])
def test_plan_rejects(change):
    assert _plan(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def _append(cache=None, k=P, k_stride=128, v=P, v_stride=128, tokens=2, positions=P, slots=P, rotary=64, cos=P, sin=P,
            rows=100):
    cache = _cache() if cache is None else cache
    return _lib.load().leafq_kv8_append(None, k, k_stride, v, v_stride, tokens, positions, slots, rotary, cos, sin, rows,
                                        ctypes.byref(cache), 0)


@pytest.mark.parametrize("change", [dict(cache=_cache(k_codes=None)), dict(cache=_cache(v_scales=None)),
                                    dict(cache=_cache(pages=0)), dict(cache=_cache(page=24)),
                                    dict(cache=_cache(kv_heads=0)), dict(cache=_cache(pages=2**26)),
                                    dict(cache=_cache(k_codes=264)), dict(k=None), dict(v=None), dict(slots=None),
                                    dict(positions=None), dict(tokens=-1), dict(tokens=2**31), dict(k_stride=127),
                                    dict(v_stride=130), dict(k_stride=64), dict(k=ODD), dict(v=ODD), dict(rotary=0),
                                    dict(rotary=60), dict(rotary=72), dict(cos=None), dict(sin=ODD), dict(rows=0)])
def test_append_rejects(change):
    assert _append(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def _attend(cache=None, step=None, q=P, stride=256, heads=4, rotary=0, cos=None, sin=None, rows=0, scale=0.125, out=P,
            workspace=P, nbytes=1 << 40):
    cache, step = _cache() if cache is None else cache, _step() if step is None else step
    return _lib.load().leafq_kv8_attention(None, q, stride, heads, rotary, cos, sin, rows, ctypes.byref(cache),
                                           ctypes.byref(step), scale, out, workspace, nbytes, 0)


@pytest.mark.parametrize("change", [dict(cache=_cache(page=8)), dict(step=_step(tokens=-1)), dict(step=_step(requests=-1)),
                                    dict(step=_step(max_tokens=-1)), dict(step=_step(max_pages=-1)),
                                    dict(step=_step(max_pages=2**31 // 64)), dict(step=_step(context=None)),
                                    dict(step=_step(lengths=None)), dict(step=_step(token_offsets=None)),
                                    dict(step=_step(page_offsets=None)), dict(step=_step(table=None)), dict(heads=0),
                                    dict(heads=5), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                    dict(scale=float("inf")), dict(q=None), dict(out=None), dict(q=ODD), dict(out=ODD),
                                    dict(stride=255), dict(stride=258), dict(rotary=64), dict(rotary=72, cos=P, sin=P, rows=9)])
def test_attention_rejects(change):
    assert _attend(**change) == _lib.LEAFQ_ERR_INVALID
    assert _lib.load().leafq_last_error()


def test_unsupported_head_sizes():
    for dim in (16, 48, 80, 160, 256):
        assert _append(cache=_cache(dim=dim), k_stride=1024, v_stride=1024) == _lib.LEAFQ_ERR_UNSUPPORTED
        assert _attend(cache=_cache(dim=dim), stride=4096) == _lib.LEAFQ_ERR_UNSUPPORTED


def test_empty_calls_are_no_ops():
    assert _append(tokens=0, k=None, v=None, slots=None) == 0
    assert _attend(step=_step(tokens=0), q=None, out=None) == 0
    assert _attend(step=_step(requests=0), q=None, out=None) == 0


def test_python_refuses_what_it_cannot_pass_on():
    f = lambda *s: torch.zeros(s)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(lq.LeafError, match="CUDA"):
        lq.Kv8Cache(f(2, 1, 16, 32).to(torch.int8), f(2, 1, 16, 32).to(torch.int8), f(2, 1), f(2, 1))
    with pytest.raises(lq.LeafError, match="block table"):
        lq.Kv8Plan(i(2), i(2), i(3), i(3), i(2), 2, 1)
    with pytest.raises(lq.LeafError, match="int32 CUDA"):
        lq.kv8_plan(i(2), i(2), i(2, 3), i(4), i(1), 16, 2)


def test_workspace_that_grows_keeps_what_a_graph_may_hold():
    workspace = lq.Kv8Workspace("cpu")
    small = workspace.get(64)
    kept, address = weakref.ref(small), small.data_ptr()
    del small
    assert workspace.get(4096).numel() == 4096
    assert kept() is not None and kept().data_ptr() == address and kept().numel() == 64
    assert workspace.get(64).numel() == 4096


class _Host:
    """Stand-ins for a cache and a plan in host memory: what the Python layer does before and around a C call, without one."""

    def __init__(self, monkeypatch, dim=32, requests=2, tokens=3):
        self.cache = types.SimpleNamespace(index=-1, device=torch.device("cpu"), dim=dim, kv_heads=1, width=dim, page=16,
                                           ref=None)
        self.plan = types.SimpleNamespace(index=-1, tokens=tokens, max_tokens=tokens, page=16, ref=None)
        self.rows = torch.zeros((tokens, dim))
        self.calls = []
        monkeypatch.setattr(kv8, "_raw_stream", lambda index: 1000 + index)
        monkeypatch.setattr(kv8, "_current_device", lambda: -1, raising=False)
        for name in ("leafq_kv8_plan", "leafq_kv8_append", "leafq_kv8_attention"):
            monkeypatch.setattr(_lib.load(), name, lambda *args, name=name: self.called(name, args))

    def called(self, name, args):
        self.calls.append((name, args))
        return 0


def test_attention_holds_its_own_workspace_until_the_call_has_returned(monkeypatch):
    host, made, alive = _Host(monkeypatch), [], []

    class Watched(lq.Kv8Workspace):
        def get(self, nbytes):
            buffer = super().get(nbytes)
            made.append(weakref.ref(buffer))
            return buffer

    monkeypatch.setattr(kv8, "Kv8Workspace", Watched)
    monkeypatch.setattr(_lib.load(), "leafq_kv8_attention", lambda *args: alive.append(made[-1]() is not None) or 0)
    lq.kv8_attention(host.rows, host.cache, host.plan, 1.0)
    assert alive == [True]


def _plan_tensors(requests=2, pages=3):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dict(context=i(requests), new_tokens=i(requests), table=i(requests, pages), free_pages=i(4), taken=i(1))


@pytest.mark.parametrize("current", [0, 1])
def test_calls_are_made_on_their_tensors_device(monkeypatch, current):
    # Tensors of device 1, with 0 or 1 current: the launch is 1's either way, and what was current is so again.
    host, devices = _Host(monkeypatch), [current]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            devices.append(self.index)

        def __exit__(self, *error):
            devices.pop()

    monkeypatch.setattr(kv8, "_current_device", lambda: devices[-1], raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    seen = []
    monkeypatch.setattr(host, "called", lambda name, args: seen.append((name, devices[-1], args[0])) or 0)
    for name in ("_check_i32", "_check_rows"):
        monkeypatch.setattr(kv8, name, lambda *a, **k: 0)
    host.cache.index = host.plan.index = 1
    workspace = types.SimpleNamespace(index=1, of=lambda *a: (0, 0))
    tensors = _plan_tensors()
    plan = types.SimpleNamespace(context=tensors["context"], table=tensors["table"], tokens=3, max_tokens=3, page=16,
                                 inputs=(0, 0, 3), outputs=(0,) * 6, index=1)
    lq.kv8_plan(**tensors, page=16, tokens=3, out=plan)
    lq.kv8_append(host.rows, host.rows, host.cache, torch.zeros(3, dtype=torch.int32))
    out = types.SimpleNamespace(get_device=lambda: 1, dtype=torch.float32, is_contiguous=lambda: True, shape=host.rows.shape,
                                data_ptr=lambda: 0)
    lq.kv8_attention(host.rows, host.cache, host.plan, 1.0, out=out, workspace=workspace)
    assert seen == [("leafq_kv8_plan", 1, 1001), ("leafq_kv8_append", 1, 1001), ("leafq_kv8_attention", 1, 1001)]
    assert devices == [current]


def test_attention_refuses_a_workspace_of_another_device(monkeypatch):
    host = _Host(monkeypatch)
    away = types.SimpleNamespace(index=0, of=lambda *a: (256, 256))
    with pytest.raises(lq.LeafError, match="workspace is on another device"):
        lq.kv8_attention(host.rows, host.cache, host.plan, 1.0, workspace=away)
    assert not host.calls
    here = lq.Kv8Workspace("cpu")
    lq.kv8_attention(host.rows, host.cache, host.plan, 1.0, workspace=here)
    assert here.index == -1 and here.device == here.buffer.device and len(host.calls) == 1


@pytest.mark.gpu
def test_workspace_keeps_the_device_that_it_was_made_on(cuda_device):
    workspace = lq.Kv8Workspace()
    assert workspace.device == torch.device("cuda", workspace.index) == workspace.get(64).device


@pytest.mark.parametrize("output,given", [("after", "taken"), ("lengths", "context"), ("lengths", "new"), ("slots", "table"),
                                          ("positions", "free"), ("token_offsets", "taken"), ("page_offsets", "context")])
def test_plan_rejects_outputs_that_overlap_its_inputs(output, given):
    # 3 requests, 3 tokens, 4 pages a row, 8 free pages, each array 256 bytes from the next.
    names = ("context", "new", "table", "free", "taken", "lengths", "token_offsets", "page_offsets", "positions", "slots", "after")
    place = {name: 4096 + 256 * i for i, name in enumerate(names)}
    place[output] = place[given]
    assert _plan(**{name: ctypes.c_void_p(at) for name, at in place.items()}) == _lib.LEAFQ_ERR_INVALID
    assert b"overlap" in _lib.load().leafq_last_error()
    # The last value of the input is as bad as the first.
    place[output] = place[given] + 4 * ({"context": 3, "new": 3, "table": 12, "free": 8, "taken": 1}[given] - 1)
    place[output] -= place[output] % 16 if output in ("positions", "slots") else 0
    assert _plan(**{name: ctypes.c_void_p(at) for name, at in place.items()}) == _lib.LEAFQ_ERR_INVALID
    assert b"overlap" in _lib.load().leafq_last_error()


def test_attention_refuses_a_plan_of_other_pages(monkeypatch):
    host = _Host(monkeypatch)
    host.plan.page = 64
    with pytest.raises(lq.LeafError, match="pages of 64 tokens, the cache of 16"):
        lq.kv8_attention(host.rows, host.cache, host.plan, 1.0)
    assert not host.calls
    for page in (16, None):  # None: a plan that its caller made and did not say
        host.plan.page = page
        lq.kv8_attention(host.rows, host.cache, host.plan, 1.0)
    assert len(host.calls) == 2


@pytest.mark.gpu
def test_plan_remembers_its_pages(cuda_device):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    context, table, free = i(2), i(2, 8), torch.arange(16, dtype=torch.int32, device="cuda")
    plan = lq.kv8_plan(context, i(2) + 20, table, free, i(1), 16, 40, max_tokens=20)
    assert plan.page == 16
    cache, q = lq.Kv8Cache.empty(16, 1, 64, 32), torch.zeros((40, 32), device="cuda")
    with pytest.raises(lq.LeafError, match="pages of 16 tokens"):
        lq.kv8_attention(q, cache, plan, 1.0)
    assert lq.kv8_plan(context, i(2) + 20, table, free, i(1), 64, 40, max_tokens=20, out=plan).page == 64
    rows = torch.ones((40, 32), device="cuda")
    lq.kv8_append(rows, rows, cache, plan.slots)
    assert torch.equal(lq.kv8_attention(q, cache, plan, 1.0), torch.ones_like(q))
    assert lq.Kv8Plan(context, plan.lengths, plan.token_offsets, plan.page_offsets, table, 40, 20).page is None
