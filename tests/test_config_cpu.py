"""The order of a config's fields is part of its interface (they may be given by place): new ones come last."""
from dataclasses import fields

from r9700_stack_b200.models.config import HybridConfig


def test_the_attention_window_comes_after_the_fields_that_were_there():
    names = [f.name for f in fields(HybridConfig)]
    first = ["qsa_topk", "qsa_heads", "hc_streams", "init_std", "tie_embeddings", "mtp_layers", "drafter", "draft_block"]
    at = names.index("qsa_topk")
    assert names[at: at + len(first)] == first
    assert {"attn_window", "attn_sinks"} <= set(names[at + len(first):])
