"""Attention of one sequence's queries to another's keys and values (an encoder's states), forward and backward."""
from .kernel import cross_attention, cross_attention_reference

__all__ = ["cross_attention", "cross_attention_reference"]
