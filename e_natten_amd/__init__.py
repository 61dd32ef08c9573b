"""Fused 2D neighborhood attention for AMD MI355X (gfx950).

Drop-in for the entry points of the reference package (e_natten/__init__.py:1):
``from e_natten_amd import natten1d, natten2d``.  For sequences that grow: ``rotary``,
``cache_append`` and ``cache_attention``; for pages that several of them share: ``cache_fork``,
``cache_reserve``, ``cache_copy`` and ``cache_compact``.
"""
from .ops import Natten1d, Natten2d, kernel_path, natten1d, natten2d
from .pages import cache_compact, cache_copy, cache_fork, cache_reserve
from .sequence import cache_append, cache_attention, rotary, rotary_axes, rotary_frequencies

__all__ = ["Natten1d", "Natten2d", "natten1d", "natten2d", "kernel_path", "rotary",
           "rotary_axes", "rotary_frequencies", "cache_append", "cache_attention",
           "cache_fork", "cache_reserve", "cache_copy", "cache_compact"]
