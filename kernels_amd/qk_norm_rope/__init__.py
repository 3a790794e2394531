"""Norms of queries and keys for each head and their rotation by position, what comes before attention, forward and backward."""
from .kernel import qk_norm_rope, qk_norm_rope_reference

__all__ = ["qk_norm_rope", "qk_norm_rope_reference"]
