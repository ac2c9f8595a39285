"""Paged INT8 KV cache: the operators of include/leafq.h's ``leafq_kv8_*``.

A pool of pages holds the keys and values of many requests as INT8 codes with
one scale per page and kv head.  One step of a batch is ``kv8_plan`` (pages and
slots from the request lengths, on the device), then per layer ``kv8_append``
(rotate, quantise, write) and ``kv8_attention``.  The reference keeps an fp32
cache per sequence (kv_cache.cpp:21-59); this one holds a quarter of its bytes
and lets requests of different lengths share memory, at the rounding of 8 bits.

``Kv8Cache``, ``Kv8Plan`` and ``Kv8Workspace`` are handles a serving loop makes
once and keeps; the calls only enqueue work on the current stream.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import LEAFQ_FLAG_PDL, LeafError, check, load

PAGE_SIZES = (16, 32, 64, 128)
HEAD_SIZES = (32, 64, 96, 128)


_F32, _I32 = torch.float32, torch.int32
_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle, without an object around it
_current_device = torch._C._cuda_getDevice


def _fail(message: str) -> None:
    raise LeafError(_lib.LEAFQ_ERR_INVALID, message)


def _need(ok: bool, message: str) -> None:
    if not ok:
        _fail(message)


# The calls sit in a decode loop, a few microseconds each: the checks below ask
# each tensor as little as they can and build their messages only to fail.  The
# library launches on the current device: a call whose tensors are on another
# is made again with that one current.
# index: of the CUDA device they have to be on (a tensor elsewhere has -1).
def _check_i32(t: torch.Tensor, name: str, numel: Optional[int] = None, index: Optional[int] = None) -> None:
    if not (t.dtype is _I32 and t.is_contiguous() and (t.is_cuda if index is None else t.get_device() == index)):
        _fail(f"{name} must be a contiguous int32 CUDA tensor, on the others' device")
    if numel is not None and t.numel() != numel:
        _fail(f"{name} must hold {numel} values")


def _check_rows(t: torch.Tensor, name: str, width: int, index: int) -> int:
    """fp32 [tokens, width] rows, contiguous in themselves (columns of a wider
    matrix are).  Returns their stride."""
    shape = t.shape
    if not (t.get_device() == index and t.dtype is _F32 and len(shape) == 2 and shape[1] == width):
        _fail(f"{name} must be float32 [tokens, {width}] on the cache's CUDA device")
    stride, inner = t.stride()
    if shape[0] != 0 and (inner != 1 or (stride < width and shape[0] != 1)):
        _fail(f"the rows of {name} must be contiguous and must not overlap")
    return stride


def _rope_args(rope, dim: int, index: int):
    """(rotary_dim, cos, sin, rows) for the C call."""
    if rope is None:
        return 0, None, None, 0
    cos, sin = rope
    shape = cos.shape
    if not (cos.get_device() == index and sin.get_device() == index and cos.dtype is _F32 and sin.dtype is _F32 and
            len(shape) == 2 and sin.shape == shape and cos.is_contiguous() and sin.is_contiguous()):
        _fail("rope tables must be two contiguous float32 [positions, rotary_dim / 2] tensors on the cache's CUDA device")
    if 2 * shape[1] > dim:
        _fail("rope tables are wider than the head")
    return 2 * shape[1], cos.data_ptr(), sin.data_ptr(), shape[0]


class Kv8Cache:
    """One layer's pool: int8 ``k`` and ``v`` [pages, kv_heads, page, dim] and
    float32 ``k_scale`` and ``v_scale`` [pages, kv_heads]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        _need(k.dim() == 4 and k.shape == v.shape, "codes must be two [pages, kv_heads, page, dim] tensors")
        self.pages, self.kv_heads, self.page, self.dim = k.shape
        for t, name in ((k, "key codes"), (v, "value codes")):
            _need(t.is_cuda and t.dtype == torch.int8 and t.is_contiguous(), f"{name} must be contiguous int8 CUDA tensors")
        for t, name in ((k_scale, "key scales"), (v_scale, "value scales")):
            _need(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() and
                  tuple(t.shape) == (self.pages, self.kv_heads), f"{name} must be contiguous float32 [pages, kv_heads]")
        _need(all(t.device == k.device for t in (v, k_scale, v_scale)), "codes and scales must be on one device")
        _need(self.page in PAGE_SIZES, f"pages hold {PAGE_SIZES} tokens")
        _need(self.dim in HEAD_SIZES, f"head sizes are {HEAD_SIZES}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.index, self.width = k.device, k.device.index, self.kv_heads * self.dim
        self.desc = _lib.Kv8CacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self.pages,
                                      self.page, self.kv_heads, self.dim)
        self.ref = ctypes.byref(self.desc)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page: int, dim: int, device="cuda") -> "Kv8Cache":
        """An uninitialised pool (a page's contents count only once written)."""
        codes = [torch.empty((pages, kv_heads, page, dim), dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.empty((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)


class Kv8Plan:
    """The arrays of one step: ``context`` and ``lengths`` [requests] (cached
    tokens before and after), ``token_offsets`` and ``page_offsets``
    [requests + 1], ``table`` [requests, max_pages], and, from ``kv8_plan``,
    ``positions`` and ``slots`` [tokens] and ``taken``.  ``tokens`` and
    ``max_tokens`` are the host's bounds: the rows of the step, and any one
    request's new tokens; ``page``, where it is given, the tokens of a page,
    which the cache's have to be."""

    def __init__(self, context, lengths, token_offsets, page_offsets, table, tokens: int, max_tokens: int,
                 positions=None, slots=None, taken=None, page: Optional[int] = None):
        _need(table.dim() == 2, "the block table must be [requests, max_pages]")
        requests, device = table.shape[0], table.device
        _check_i32(table, "the block table")
        _check_i32(context, "context", requests, device.index)
        _check_i32(lengths, "lengths", requests, device.index)
        _check_i32(token_offsets, "token_offsets", requests + 1, device.index)
        _check_i32(page_offsets, "page_offsets", requests + 1, device.index)
        _need(tokens >= 0 and max_tokens >= 0, "token counts must not be negative")
        self.context, self.lengths, self.table = context, lengths, table
        self.token_offsets, self.page_offsets = token_offsets, page_offsets
        self.positions, self.slots, self.taken = positions, slots, taken
        self.requests, self.tokens, self.max_tokens, self.device = requests, int(tokens), int(max_tokens), device
        self.index, self.page = device.index, page
        self.inputs = self.outputs = None  # addresses, of a plan that kv8_plan made
        self.desc = _lib.Kv8StepDesc(context.data_ptr(), lengths.data_ptr(), token_offsets.data_ptr(),
                                     page_offsets.data_ptr(), table.data_ptr(), table.shape[1], self.tokens,
                                     self.max_tokens, requests)
        self.ref = ctypes.byref(self.desc)

    def bound(self, max_tokens: int) -> None:
        """Another bound on any one request's new tokens, for the calls to come."""
        _need(max_tokens >= 0, "token counts must not be negative")
        self.max_tokens = self.desc.max_tokens = int(max_tokens)


class Kv8Workspace:
    """Device scratch of ``kv8_attention``, zeroed when it grows.  Reuse it
    across calls on one stream.  A buffer that was outgrown lives as long as the
    handle: a graph captured with it holds its address, and so do calls that
    have not run yet.  Keep the handle as long as the graph."""

    def __init__(self, device="cuda"):
        self.buffer = torch.empty(0, dtype=torch.uint8, device=device)
        self.device, self.index = self.buffer.device, self.buffer.get_device()
        self.outgrown: list = []
        self.sizes: dict = {}

    def get(self, nbytes: int) -> torch.Tensor:
        if nbytes > self.buffer.numel():
            self.outgrown.append(self.buffer)
            self.buffer = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
        return self.buffer

    def of(self, max_tokens: int, heads: int, kv_heads: int, dim: int):
        """(address, bytes) for a geometry."""
        key = (max_tokens, heads, kv_heads, dim)
        need = self.sizes.get(key)
        if need is None:
            need = self.sizes[key] = load().leafq_kv8_attention_workspace_bytes(*key)
        return self.get(need).data_ptr(), need


def kv8_plan(context: torch.Tensor, new_tokens: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
             taken: torch.Tensor, page: int, tokens: int, max_tokens: Optional[int] = None,
             out: Optional[Kv8Plan] = None, flags: int = LEAFQ_FLAG_PDL) -> Kv8Plan:
    """Pages and slots of a step.  Request s holds context[s] tokens and brings
    new_tokens[s]; the pages they need are taken from free_pages[taken:] in
    request order and written into its row of ``table`` (in place).  A request
    that does not fit its row or the free pages is refused: slots -1 and
    lengths[s] == context[s].  tokens: the step's rows, at least the sum of
    new_tokens (the rest get slot -1); max_tokens: a bound on any request's new
    tokens (default: tokens).  ``taken`` is only read, the new count is the
    plan's ``taken`` (copy it back for the next step: outputs that overlap the
    inputs are refused).  ``out``: a plan of the same buffers and rows, which is
    filled again; max_tokens may be another."""
    index = context.get_device() if out is None else out.index
    if index >= 0 and _current_device() != index:
        with torch.cuda.device(index):
            return kv8_plan(context, new_tokens, table, free_pages, taken, page, tokens, max_tokens, out, flags)
    requests = context.numel()
    most = tokens if max_tokens is None else max_tokens
    if out is not None and out.context is context and out.table is table and out.tokens == tokens and out.inputs is not None:
        plan = out
        if plan.max_tokens != most:
            plan.bound(most)
    else:
        device = context.device
        _need(out is None, "the plan to reuse is of other buffers or sizes")
        _check_i32(context, "context")
        _need(table.dim() == 2 and table.shape[0] == requests, "the block table must be [requests, max_pages]")
        sizes = (requests, requests + 1, requests + 1, 1, tokens, tokens)
        room = [-(-n // 4) * 4 for n in sizes]  # 16-byte aligned pieces
        pieces = torch.empty(sum(room), dtype=torch.int32, device=device).split(room)
        lengths, token_offsets, page_offsets, after, positions, slots = (p[:n] for p, n in zip(pieces, sizes))
        plan = Kv8Plan(context, lengths, token_offsets, page_offsets, table, tokens, most, positions, slots, after)
        plan.inputs = (context.data_ptr(), table.data_ptr(), table.shape[1])
        plan.outputs = tuple(p.data_ptr() for p in (lengths, token_offsets, page_offsets, positions, slots, after))
    _check_i32(new_tokens, "new_tokens", requests, plan.index)
    _check_i32(free_pages, "free_pages", None, plan.index)
    _check_i32(taken, "taken", 1, plan.index)
    check(load().leafq_kv8_plan(_raw_stream(plan.index), plan.inputs[0], new_tokens.data_ptr(), requests, plan.inputs[1],
                                plan.inputs[2], free_pages.data_ptr(), free_pages.numel(), taken.data_ptr(), page, tokens,
                                *plan.outputs, flags))
    plan.page = page
    return plan


def kv8_append(k: torch.Tensor, v: torch.Tensor, cache: Kv8Cache, slots: torch.Tensor,
               positions: Optional[torch.Tensor] = None, rope=None, flags: int = LEAFQ_FLAG_PDL) -> None:
    """Writes the rows of k and v (fp32 [tokens, kv_heads * dim]; columns of a
    wider matrix will do) into the cache at their slots, -1 skipping a row.
    With rope = (cos, sin) tables [positions, rotary_dim / 2] the keys are
    rotated by ``positions`` first.  A page's scale grows when a new row needs
    it, and its older codes are rounded to the new scale."""
    index = cache.index
    if _current_device() != index:
        with torch.cuda.device(index):
            return kv8_append(k, v, cache, slots, positions, rope, flags)
    k_stride = _check_rows(k, "k", cache.width, index)
    v_stride = _check_rows(v, "v", cache.width, index)
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        _fail("k and v must have the same rows")
    _check_i32(slots, "slots", tokens, index)
    rotary, cos, sin, rows = _rope_args(rope, cache.dim, index)
    where = None
    if rope is not None:
        if positions is None:
            _fail("rotation needs positions")
        _check_i32(positions, "positions", tokens, index)
        where = positions.data_ptr()
    check(load().leafq_kv8_append(_raw_stream(index), k.data_ptr(), k_stride, v.data_ptr(), v_stride, tokens, where,
                                  slots.data_ptr(), rotary, cos, sin, rows, cache.ref, flags))


def kv8_attention(q: torch.Tensor, cache: Kv8Cache, plan: Kv8Plan, scale: float, rope=None,
                  out: Optional[torch.Tensor] = None, workspace: Optional[Kv8Workspace] = None,
                  flags: int = LEAFQ_FLAG_PDL) -> torch.Tensor:
    """Causal grouped-query attention of the step's rows q (fp32
    [tokens, heads * dim]; columns of a wider matrix will do) over the cache,
    rotated by position when rope tables are given.  Returns fp32
    [tokens, heads * dim]; a row that sees no key is zero, rows past the step's
    last new token are not written."""
    index, dim, shape = cache.index, cache.dim, q.shape
    if _current_device() != index:
        with torch.cuda.device(index):
            return kv8_attention(q, cache, plan, scale, rope, out, workspace, flags)
    if len(shape) != 2 or shape[1] % dim != 0:
        _fail("q must be [tokens, heads * dim]")
    tokens, width = shape
    stride = _check_rows(q, "q", width, index)
    if tokens != plan.tokens:
        _fail("q has other rows than the plan")
    if plan.index != index:
        _fail("the plan is on another device")
    if plan.page is not None and plan.page != cache.page:
        _fail(f"the plan has pages of {plan.page} tokens, the cache of {cache.page}")
    if out is None:
        out = torch.empty_like(q)  # contiguous, as q's rows do not overlap
    elif not (out.get_device() == index and out.dtype is _F32 and out.is_contiguous() and out.shape == shape):
        _fail("out must be contiguous float32 of q's shape, on its device")
    rotary, cos, sin, rows = _rope_args(rope, dim, index)
    heads = width // dim
    if workspace is None:
        workspace = Kv8Workspace(cache.device)  # in a name of its own, until the launch is enqueued
    elif workspace.index != index:
        _fail("the workspace is on another device")
    address, need = workspace.of(plan.max_tokens, heads, cache.kv_heads, dim)
    check(load().leafq_kv8_attention(_raw_stream(index), q.data_ptr(), stride, heads, rotary, cos, sin, rows, cache.ref,
                                     plan.ref, scale, out.data_ptr(), address, need, flags))
    return out
