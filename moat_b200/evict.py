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

import struct

from ._lib import check, lib
from .tree import _device_index, _five, _on, _on_device, _plain, _rows, _torch, _Workspaces

_ws = _Workspaces()
_sizes = {}  # workspace bytes by geometry
_Args = struct.Struct("@10PN8q8i")  # the C struct mb_cache_evict_args


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
    t = _torch()
    scores_out = scores if scores_out is None else scores_out
    positions_out = positions if positions_out is None else positions_out
    try:
        idx = k_cache.get_device()
        full, dt, i32, f32 = tuple(k_cache.shape), k_cache.dtype, t.int32, t.float32
        layers = full[0] if len(full) == 5 else 1
        T, Hkv, Lmax, d = full[-4:]
        rows, one = full[:-1], (T,)
        sk, sv = k_cache.stride(), v_cache.stride()
        fine = (idx >= 0 and idx == v_cache.get_device() == scores.get_device() == positions.get_device()
                == lens.get_device() == next_pos.get_device() == scores_out.get_device() == positions_out.get_device()
                and 4 <= len(full) <= 5 and min(full) >= 1 and v_cache.shape == full and dt is v_cache.dtype
                and dt.itemsize == 2 and (sk[-1] == sv[-1] == 1 or d == 1)
                and f32 is scores.dtype is scores_out.dtype
                and i32 is positions.dtype is positions_out.dtype is lens.dtype is next_pos.dtype
                and scores.shape == rows and scores_out.shape == rows and positions.shape == rows
                and positions_out.shape == rows and lens.shape == one and next_pos.shape == one
                and scores.is_contiguous() and scores_out.is_contiguous() and positions.is_contiguous()
                and positions_out.is_contiguous() and lens.is_contiguous() and next_pos.is_contiguous())
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _check_evict(k_cache, v_cache, scores, positions, lens, next_pos, scores_out, positions_out)
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if not (budget >= 1 and recent >= 0 and sinks >= 0 and recent + sinks <= budget):
        raise ValueError("budget must be positive and hold the recent rows and the sinks")
    ps, pp, pso, ppo = scores.data_ptr(), positions.data_ptr(), scores_out.data_ptr(), positions_out.data_ptr()
    if (pso == ps) != (ppo == pp):
        raise ValueError("scores and positions are both updated in place, or neither")
    new_lens = t.empty_like(lens)
    L = lib()
    geometry = (layers, T, Hkv, Lmax, budget)
    nbytes = _sizes.get(geometry)
    if nbytes is None:
        nbytes = _sizes[geometry] = int(L.mb_cache_evict_workspace_size(*geometry))
    lead = () if len(full) == 5 else (0,)

    def call(st):
        ws = _ws.get(idx, st, nbytes)
        return L.mb_cache_evict(_Args.pack(
            k_cache.data_ptr(), v_cache.data_ptr(), ps, pp, pso, ppo, lens.data_ptr(), next_pos.data_ptr(),
            new_lens.data_ptr(), ws[0], ws[1], *lead, *sk[:-1], *lead, *sv[:-1], layers, T, Hkv, Lmax, d, budget, recent,
            sinks), st)

    rc = _on(idx, call)
    if rc != 0:
        check(rc, "mb_cache_evict")
    return scores_out, positions_out, new_lens


__all__ = ["evict_cache"]
