"""Verification of drafted tokens (include/leafq.h, leafq_verify_drafts).

A step that checks drafts runs the model over every row of a request's tree, the
token that is certain first, and asks the target's logits which of the drafts
stand: with random numbers from the caller, the tokens that come out follow the
target's distribution whatever proposed the drafts.  The reference decodes one
token a step (main_decoder.cpp:95-113).
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import LEAFQ_FLAG_PDL, check, load
from .kv8 import _F32, _I32, Kv8Plan, _check_i32, _current_device, _fail, _raw_stream


class Verdict:
    """Which rows stand: ``path`` [requests, max_tokens], the rows of the walk
    from each request's row 0; ``tokens`` [requests, max_tokens], the token behind
    each of them (both end with -1s); ``kept`` [requests], how many there are;
    ``next`` [requests], the last of the tokens."""

    def __init__(self, requests: int, max_tokens: int, device):
        self.path, self.tokens = (torch.empty((requests, max_tokens), dtype=_I32, device=device) for _ in range(2))
        self.kept, self.next = (torch.empty(requests, dtype=_I32, device=device) for _ in range(2))
        self.requests, self.max_tokens, self.index = requests, max_tokens, self.kept.get_device()
        self.address = tuple(t.data_ptr() for t in (self.path, self.tokens, self.kept, self.next))


def _check_f32(t: torch.Tensor, name: str, numel: int, index: int) -> None:
    if not (t.dtype is _F32 and t.is_contiguous() and t.get_device() == index and t.numel() == numel):
        _fail(f"{name} must be {numel} contiguous float32 values on the plan's CUDA device")


def _check_rows(t: torch.Tensor, name: str, tokens: int, index: int) -> int:
    """float32 [tokens, vocab], each row contiguous.  Returns the rows' stride."""
    shape = t.shape
    if not (t.dtype is _F32 and t.get_device() == index and len(shape) == 2 and shape[0] == tokens):
        _fail(f"{name} must be float32 [tokens, vocab] on the plan's CUDA device")
    stride, inner = t.stride()
    if (inner != 1 and shape[1] > 1) or (stride < shape[1] and tokens > 1):
        _fail(f"the rows of {name} must be contiguous and must not overlap")
    return stride


def verify_drafts(logits: torch.Tensor, ids: torch.Tensor, parents: torch.Tensor, plan: Kv8Plan, accept: torch.Tensor,
                  sample: torch.Tensor, temperature: torch.Tensor, draft_probs: Optional[torch.Tensor] = None,
                  out: Optional[Verdict] = None, flags: int = LEAFQ_FLAG_PDL) -> Verdict:
    """Walks every request's tree from its row 0 and keeps the drafts that the
    target takes.  logits (float32 [tokens, vocab]; rows may be further apart)
    are the target's behind each row; ids and parents (int32 [tokens]) the rows'
    tokens and trees, as kv8_tree has them.  A child c of row u is taken when
    accept[c] * q < p of its token, p = softmax(logits[u] / temperature) less what
    its rejected siblings took, q = draft_probs[u] (float32 [tokens, vocab]) or 1
    for drafts that were not drawn.  The token behind the last row is drawn by
    sample from what p then is.  accept [tokens] and sample [requests] are uniform
    in [0, 1); temperature [requests] of 0 is greedy.  ``out``: a verdict of the same
    sizes, which is filled again (its tensors may not be inputs of the call)."""
    index = plan.index
    if _current_device() != index:
        with torch.cuda.device(index):
            return verify_drafts(logits, ids, parents, plan, accept, sample, temperature, draft_probs, out, flags)
    tokens, requests = plan.tokens, plan.requests
    stride = _check_rows(logits, "logits", tokens, index)
    vocab = logits.shape[1]
    _check_i32(ids, "ids", tokens, index)
    _check_i32(parents, "parents", tokens, index)
    _check_f32(accept, "accept", tokens, index)
    _check_f32(sample, "sample", requests, index)
    _check_f32(temperature, "temperature", requests, index)
    probs = probs_stride = 0
    if draft_probs is not None:
        probs_stride = _check_rows(draft_probs, "draft_probs", tokens, index)
        if draft_probs.shape[1] != vocab:
            _fail("draft_probs must have the logits' shape")
        probs = draft_probs.data_ptr()
    if out is None:
        out = Verdict(requests, plan.max_tokens, plan.device)
    elif out.requests != requests or out.max_tokens != plan.max_tokens or out.index != index:
        _fail("the verdict to reuse is of other sizes, or on another device")
    check(load().leafq_verify_drafts(_raw_stream(index), logits.data_ptr(), stride, vocab, ids.data_ptr(), parents.data_ptr(),
                                     plan.token_offsets.data_ptr(), requests, tokens, plan.max_tokens, accept.data_ptr(),
                                     sample.data_ptr(), temperature.data_ptr(), probs or None, probs_stride, *out.address,
                                     flags))
    return out
