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

import ctypes

from . import _lib
from ._lib import check, lib, stream_of
from .tree import _five, _need, _on_device, _plain

_pool = _lib.WorkspacePool()
_Strides8 = ctypes.c_int64 * 8


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
    t = _lib.require_cuda()
    if not isinstance(k_cache, t.Tensor):
        raise TypeError("k_cache must be a torch CUDA tensor")
    dev = k_cache.device
    scores_out = scores if scores_out is None else scores_out
    positions_out = positions if positions_out is None else positions_out
    _on_device(t, dev, k_cache=k_cache, v_cache=v_cache, scores=scores, positions=positions, lens=lens,
               next_pos=next_pos, scores_out=scores_out, positions_out=positions_out)
    kc, vc = _five(k_cache, "k_cache"), _five(v_cache, "v_cache")
    layers, T, Hkv, Lmax, d = kc.shape
    _need(min(layers, T, Hkv, Lmax, d) >= 1, "the caches must not be empty")
    _need(vc.shape == kc.shape, "k_cache and v_cache must have one shape")
    strides = []
    for x in (kc, vc):
        st = x.stride()
        if x.dtype is not kc.dtype or x.element_size() != 2 or (st[4] != 1 and d > 1):
            raise ValueError("the caches must share one 16-bit dtype and be contiguous along the head dim")
        strides += st[:4]
    full = tuple(k_cache.shape[:-1])
    for x, dtype, n in ((scores, t.float32, "scores"), (scores_out, t.float32, "scores_out"),
                        (positions, t.int32, "positions"), (positions_out, t.int32, "positions_out")):
        _plain(x, full, dtype, n)
    _plain(lens, (T,), t.int32, "lens")
    _plain(next_pos, (T,), t.int32, "next_pos")
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    _need(budget >= 1 and recent >= 0 and sinks >= 0 and recent + sinks <= budget,
          "budget must be positive and hold the recent rows and the sinks")
    _need((scores_out.data_ptr() == scores.data_ptr()) == (positions_out.data_ptr() == positions.data_ptr()),
          "scores and positions are both updated in place, or neither")
    new_lens = t.empty_like(lens)
    L = lib()
    with t.cuda.device(dev):
        st = stream_of(dev)
        ws = _pool.get(dev, st, int(L.mb_cache_evict_workspace_size(layers, T, Hkv, Lmax, budget)))
        rc = L.mb_cache_evict(kc.data_ptr(), vc.data_ptr(), _Strides8(*strides), scores.data_ptr(),
                              positions.data_ptr(), scores_out.data_ptr(), positions_out.data_ptr(), lens.data_ptr(),
                              next_pos.data_ptr(), new_lens.data_ptr(), layers, T, Hkv, Lmax, d, budget, recent, sinks,
                              ws.data_ptr(), ws.numel(), st)
    if rc != 0:
        check(rc, "mb_cache_evict")
    return scores_out, positions_out, new_lens


__all__ = ["evict_cache"]
