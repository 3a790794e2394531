"""Streaming attention for serving: the newest tokens of every sequence over a cache of keys and values in pages."""
from .kernel import paged_append, paged_attention, paged_attention_reference

__all__ = ["paged_attention", "paged_append", "paged_attention_reference"]
