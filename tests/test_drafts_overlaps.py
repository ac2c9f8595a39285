"""Calls that check drafted tokens refuse outputs that share memory with what others of their blocks still read,
on the host, before touching a device."""
import ctypes

import pytest

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
