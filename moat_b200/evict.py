"""Eviction from a KV cache by accumulated attention weight.

A long rollout outgrows its cache. ``evict_cache`` brings every (layer, trace, KV head)
back to ``budget`` rows: the recent ones, the first positions (``sinks``) and those with
the largest ``scores``, the attention weight that ``moat_b200.tree.tree_attention`` sums up
per row. Attention does not depend on the order of a cache's rows (a key carries its
rotary position), so the rows that stay are not shifted: each one beyond the budget moves
into the place of one that leaves, and ``positions`` says which position a row holds.
The reference keeps every row until its cache overflows (``batch_generator.py:79-107``).
"""

from __future__ import annotations

from . import _lib
from .tree import _device_index, _done, _five, _on_device, _own_places, _plain, _rows, _torch


def _check_evict(k_cache, v_cache, scores, positions, lens, next_pos, scores_out, positions_out):
    t = _torch()
    idx = _device_index(k_cache, "k_cache")
    _on_device(idx, v_cache=v_cache, scores=scores, positions=positions, lens=lens, next_pos=next_pos,
               scores_out=scores_out, positions_out=positions_out)
    kc, vc = _five(k_cache, "k_cache"), _five(v_cache, "v_cache")
    if min(kc.shape) < 1:
        raise ValueError("the caches must not be empty")
    if vc.shape != kc.shape:
        raise ValueError("k_cache and v_cache must have one shape")
    what = "the caches must share one 16-bit dtype and be contiguous along the head dim"
    if kc.element_size() != 2:
        raise ValueError(what)
    _rows(kc.dtype, what, kc, vc)
    _own_places(k_cache=kc, v_cache=vc)
    full = k_cache.shape[:-1]
    _plain(scores, full, t.float32, "scores")
    _plain(scores_out, full, t.float32, "scores_out")
    _plain(positions, full, t.int32, "positions")
    _plain(positions_out, full, t.int32, "positions_out")
    _plain(lens, (kc.shape[1],), t.int32, "lens")
    _plain(next_pos, (kc.shape[1],), t.int32, "next_pos")


def evict_cache(k_cache, v_cache, scores, positions, lens, next_pos, budget: int, *, recent: int, sinks: int = 0,
                scores_out=None, positions_out=None):
    """Keep ``min(lens[t], budget)`` rows of every cache.

    * ``k_cache`` / ``v_cache [layers, T, Hkv, Lmax, d]`` (or without the layer axis), any
      16-bit dtype, last axis contiguous: rows move in place.
    * ``scores`` float32 and ``positions`` int32 ``[layers, T, Hkv, Lmax]``, contiguous.
      ``scores_out`` / ``positions_out`` (default: in place) get the kept rows' values and
      keep what they hold beyond them.
    * ``lens`` int32 ``[T]``, ``next_pos`` int32 ``[T]`` (the position of the next token).

    A row is guarded if its position is at least ``next_pos[t] - recent`` or below
    ``sinks`` (``recent + sinks <= budget``). Guarded rows rank alike, above all others, then
    larger scores; equal ones by lowest row; a NaN ranks below everything. With at most
    ``budget`` rows nothing moves. Kept row ``r < budget`` stays at ``r``; the j-th kept row
    at or beyond the budget goes to the j-th row below it that leaves.

    Returns ``(scores_out, positions_out, new_lens)``.
    """
    scores_out = scores if scores_out is None else scores_out
    positions_out = positions if positions_out is None else positions_out
    r = _lib.bind().evict(k_cache, v_cache, scores, positions, lens, next_pos, scores_out, positions_out, int(budget),
                          int(recent), int(sinks))
    if r is None or type(r) is int:
        _done(r, "mb_cache_evict", _check_evict, k_cache, v_cache, scores, positions, lens, next_pos, scores_out,
              positions_out)
    return r


__all__ = ["evict_cache"]
