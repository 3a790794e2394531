"""Streaming attention for serving: the newest tokens of every sequence, or trees of drafted ones, over a cache of keys and values in pages."""
from .kernel import (
    paged_append,
    paged_append_rope,
    paged_attention,
    paged_attention_reference,
    paged_keep,
    paged_tree_attention,
    paged_tree_attention_reference,
)

__all__ = ["paged_attention", "paged_append", "paged_attention_reference", "paged_append_rope", "paged_tree_attention", "paged_keep",
           "paged_tree_attention_reference"]
