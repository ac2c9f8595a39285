"""leaf_b200: B200-native (sm_100a) quantised-linear operators for Leaf.

The hot path -- per-token INT8 activation quantisation, the W8A8 / W4A8 /
W4A32 decode GEMV, the W8A8 tcgen05 prefill GEMM, the dequant + bias
epilogue and the graph executor's INT8 GEMM -- runs in libleafq.so (C ABI in
include/leafq.h).  This package is the host-side mirror of the reference's
operator interface plus the N-sharded multi-GPU wrapper.  kv8 is a paged INT8 KV cache
(step plan, append, attention) for batches of requests of unlike lengths, and checks
trees of drafted tokens over it; drafts verifies them against the target's logits.
"""
from ._lib import LeafError, LEAFQ_FLAG_PDL, LEAFQ_FLAG_VNNI_ROUNDING, load
from .drafts import Verdict, verify_drafts
from .kv8 import (Kv8Cache, Kv8Layers, Kv8Plan, Kv8Released, Kv8Tree, Kv8Workspace, kv8_append, kv8_attention,
                  kv8_compact, kv8_plan, kv8_release, kv8_tree, kv8_tree_attention)
from .linear import (QuantLinearSet, QuantWeight, Workspace, gemm_i8_per_channel,
                     graph_linear, graph_quantize, linear, linear_int_q, quantize_act)

__all__ = [
    "LeafError", "LEAFQ_FLAG_PDL", "LEAFQ_FLAG_VNNI_ROUNDING", "load", "QuantLinearSet",
    "QuantWeight", "Workspace", "gemm_i8_per_channel", "graph_linear", "graph_quantize", "linear",
    "linear_int_q", "quantize_act", "Kv8Cache", "Kv8Plan", "Kv8Workspace", "kv8_append",
    "kv8_attention", "kv8_plan", "Kv8Layers", "Kv8Released", "Kv8Tree", "Verdict", "kv8_compact",
    "kv8_release", "kv8_tree", "kv8_tree_attention", "verify_drafts",
]
