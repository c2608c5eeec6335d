"""Drafted decoding over a KV cache: attention of a tree of drafted tokens, and acceptance
of the verified tree.

A decode step can check several drafted tokens of a trace at once. The drafted tokens form
a tree of ``m <= 64`` nodes in topological order (``parents[0] = -1``: node 0 is the last
token the model chose, its keys not yet in the cache; ``0 <= parents[i] < i``; any other
parent marks padding). Their keys and values live in draft buffers ``[T, m, Hkv, d]`` until
the tree is verified; then the accepted rows are appended to the caches and the rest is
dropped, so a cache never holds a rejected row.

``tree_attention`` is exact softmax attention (the reference's PyTorch decoder,
``transformer.py:110-119``, one query per step); ``m = 1`` is its single-token step.
Grouped KV heads (``H`` a multiple of ``Hkv``) and fp16 or bf16 are taken. With ``scores``
it also keeps the accumulated attention weight of every cached row, which
``moat_b200.evict.evict_cache`` ranks rows by.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import numpy as np

from . import _lib
from ._lib import check, lib, stream_of

MAX_NODES = 64  # one bit per node in a mask

_pool = _lib.WorkspacePool()


def tree_masks(parents) -> np.ndarray:
    """Ancestors-or-self of every node as the bits of an int64: ``parents [..., m]`` (any
    sequence; a parent that is not an earlier node marks padding) -> int64 ``[..., m]``, 0
    for padding."""
    par = np.asarray(parents, dtype=np.int64)
    m = par.shape[-1] if par.ndim else 0
    if not 1 <= m <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {m}")
    flat = par.reshape(-1, m)
    out = np.zeros(flat.shape, dtype=np.uint64)
    rows = np.arange(flat.shape[0])
    for i in range(m):
        p = flat[:, i]
        above = out[rows, np.clip(p, 0, m - 1)]
        real = (p >= 0) & (p < i) & (above != 0) if i else np.full(flat.shape[0], True)
        out[:, i] = np.where(real, above * np.uint64(i > 0) | np.uint64(1 << i), np.uint64(0))
    return out.view(np.int64).reshape(par.shape)


def tree_depths(parents) -> np.ndarray:
    """Distance of every node from the root, int32 like ``parents`` (0 for padding)."""
    par = np.asarray(parents, dtype=np.int64)
    m = par.shape[-1]
    flat, masks = par.reshape(-1, m), tree_masks(par).reshape(-1, m)
    out = np.zeros(flat.shape, dtype=np.int32)
    rows = np.arange(flat.shape[0])
    for i in range(1, m):
        out[:, i] = np.where(masks[:, i] != 0, out[rows, np.clip(flat[:, i], 0, m - 1)] + 1, 0)
    return out.reshape(par.shape)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on_device(t, dev, **tensors) -> None:
    for name, x in tensors.items():
        if not isinstance(x, t.Tensor):
            raise TypeError(f"{name} must be a torch CUDA tensor")
        if not x.is_cuda or x.device != dev:
            raise ValueError(f"{name} must be on {dev}")


def _plain(x, shape, dtype, name) -> None:
    """A contiguous tensor of one shape and dtype."""
    if tuple(x.shape) != shape or x.dtype != dtype or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)}")


_Strides18 = ctypes.c_int64 * 18
_Strides16 = ctypes.c_int64 * 16


def tree_attention(q, k_cache, v_cache, lens, k_draft, v_draft, masks, *, scale=None, out=None, scores=None,
                   scores_out=None, draft_scores=None, dev_err=None):
    """Attention of every node of every trace's tree.

    * ``q [T, m, H, d]``, ``k_cache`` / ``v_cache [T, Hkv, Lmax, d]`` (the first ``lens[t]``
      rows valid), ``k_draft`` / ``v_draft [T, m, Hkv, d]``: fp16 or bf16, CUDA, the last
      axis contiguous, other strides free; ``d <= 256``.
    * ``lens`` int32 ``[T]``, ``masks`` int64 ``[T, m]`` or ``[m]`` (one tree for every
      trace): node ``i`` sees all committed rows and the nodes whose bit is set. A mask of 0
      marks padding: the node sees nothing and its output is 0.
    * ``out``: optional result ``[T, m, H, d]``; ``scale`` defaults to ``1/sqrt(d)``.
    * ``scores`` float32 ``[T, Hkv, Lmax]``: also compute, for every row, its attention
      weight summed over the nodes and the heads of its group. ``scores_out`` (default: in
      place) gets ``scores`` plus that sum in the first ``lens[t]`` rows and keeps the
      others; ``draft_scores`` float32 ``[T, Hkv, m]`` gets the sums of the draft's rows.

    * ``dev_err``: optional int32 CUDA tensor whose first word receives device error bits
      (bounded waits).

    fp32 scores, softmax and sums; one rounding at the output (and one of each unnormalised
    probability to the inputs' type before its product with V). Repeated calls give the same
    bits. Returns ``out``, or ``(out, scores_out, draft_scores)`` with ``scores``.
    """
    t = _lib.require_cuda()
    if not isinstance(q, t.Tensor):
        raise TypeError("q must be a torch CUDA tensor")
    dev = q.device
    _on_device(t, dev, q=q, k_cache=k_cache, v_cache=v_cache, lens=lens, k_draft=k_draft, v_draft=v_draft, masks=masks)
    if q.dim() != 4 or k_cache.dim() != 4:
        raise ValueError("q must be [T, m, H, d] and the caches [T, Hkv, Lmax, d]")
    T, m, H, d = q.shape
    Hkv, Lmax = k_cache.shape[1], k_cache.shape[2]
    if not 1 <= m <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {m}")
    if T < 1 or Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"{H} query heads do not divide among {Hkv} KV heads")
    if not 1 <= d <= 256:
        raise ValueError(f"head dim must be 1 to 256, got {d}")
    if k_cache.shape != (T, Hkv, Lmax, d) or v_cache.shape != (T, Hkv, Lmax, d):
        raise ValueError(f"k_cache / v_cache must be [{T}, {Hkv}, Lmax, {d}]")
    if k_draft.shape != (T, m, Hkv, d) or v_draft.shape != (T, m, Hkv, d):
        raise ValueError(f"k_draft / v_draft must be [{T}, {m}, {Hkv}, {d}]")
    dt = q.dtype
    if dt is not t.float16 and dt is not t.bfloat16:
        raise ValueError("q must be fp16 or bf16")
    _plain(lens, (T,), t.int32, "lens")
    shared = masks.dim() == 1
    _plain(masks, (m,) if shared else (T, m), t.int64, "masks")
    if out is None:
        out = t.empty((T, m, H, d), dtype=dt, device=dev)
    else:
        _on_device(t, dev, out=out)
        _need(out.shape == q.shape, f"out must be [{T}, {m}, {H}, {d}]")
    six = (q, k_cache, v_cache, k_draft, v_draft, out)
    strides = []
    for x in six:
        st = x.stride()
        if x.dtype is not dt or (st[3] != 1 and d > 1):
            raise ValueError("q, out, caches and drafts must share one dtype and be contiguous along the head dim")
        strides += st[:3]
    sc = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _need(math.isfinite(sc), "scale must be finite")
    ps = pso = pds = None
    if scores is not None:
        scores_out = scores if scores_out is None else scores_out
        if draft_scores is None:
            draft_scores = t.empty((T, Hkv, m), dtype=t.float32, device=dev)
        _on_device(t, dev, scores=scores, scores_out=scores_out, draft_scores=draft_scores)
        _plain(scores, (T, Hkv, Lmax), t.float32, "scores")
        _plain(scores_out, (T, Hkv, Lmax), t.float32, "scores_out")
        _plain(draft_scores, (T, Hkv, m), t.float32, "draft_scores")
        ps, pso, pds = scores.data_ptr(), scores_out.data_ptr(), draft_scores.data_ptr()
    else:
        _need(scores_out is None and draft_scores is None, "scores_out and draft_scores need scores")
    if dev_err is not None:
        _on_device(t, dev, dev_err=dev_err)
    L = lib()
    with t.cuda.device(dev):
        st = stream_of(dev)
        ws = _pool.get(dev, st, int(L.mb_tree_attn_workspace_size(T, m, H, Hkv, Lmax, d)))
        rc = L.mb_tree_attn(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr(), k_draft.data_ptr(),
                            v_draft.data_ptr(), masks.data_ptr(), 1 if shared else 0, out.data_ptr(),
                            _Strides18(*strides), 1 if dt is t.bfloat16 else 0, T, m, H, Hkv, Lmax, d, sc, ps, pso,
                            pds, ws.data_ptr(), ws.numel(), None if dev_err is None else dev_err.data_ptr(), st)
    if rc != 0:
        check(rc, "mb_tree_attn")
    return out if scores is None else (out, scores_out, draft_scores)


class Accepted(NamedTuple):
    """What ``accept_tree`` found, all int32 on the device."""

    path: object  # [T, m] accepted nodes from the root on, -1 after the last
    counts: object  # [T] accepted nodes (the root included)
    next_ids: object  # [T] the model's choice after the last accepted node
    lens: object  # [T] cache rows after the append
    next_pos: object  # [T] position of the next token


def _five(x, name):
    """[layers, ...] of a tensor with or without its layer axis."""
    if x.dim() == 4:
        return x.unsqueeze(0)
    if x.dim() != 5:
        raise ValueError(f"{name} must have 4 axes, or 5 with layers first")
    return x


def accept_tree(tokens, parents, target, lens, next_pos, k_cache, v_cache, k_draft, v_draft, *, scores=None,
                draft_scores=None, positions=None, dev_err=None) -> Accepted:
    """Greedy acceptance of a verified tree, and the append of its accepted rows.

    From the root, the first child whose drafted token equals the model's choice at its
    parent is accepted, and so on. ``tokens`` / ``target`` int32 ``[T, m]`` (the drafted
    tokens; the model's choice at every node), ``parents`` int32 ``[T, m]`` or ``[m]``.
    A negative token is never accepted; a trace whose root token is negative is idle
    (count 0, next id -1).

    Row ``lens[t] + j`` of the caches ``[layers, T, Hkv, Lmax, d]`` (or without the layer
    axis) gets the j-th accepted node's row of the drafts ``[layers, T, m, Hkv, d]``, in
    place; likewise ``scores`` (float32 ``[layers, T, Hkv, Lmax]``) from ``draft_scores``
    (``[layers, T, Hkv, m]``), and ``positions`` (int32, like ``scores``) gets
    ``next_pos[t] + j``. A trace without room for its accepted rows keeps its state (count
    0) and sets bit 2 of ``dev_err`` (int32 CUDA tensor, optional). 16-bit element types.
    """
    t = _lib.require_cuda()
    if not isinstance(k_cache, t.Tensor):
        raise TypeError("k_cache must be a torch CUDA tensor")
    dev = k_cache.device
    _on_device(t, dev, tokens=tokens, parents=parents, target=target, lens=lens, next_pos=next_pos, k_cache=k_cache,
               v_cache=v_cache, k_draft=k_draft, v_draft=v_draft)
    kc, vc, kd, vd = (_five(x, n) for x, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (k_draft, "k_draft"),
                                               (v_draft, "v_draft")))
    layers, T, Hkv, Lmax, d = kc.shape
    m = kd.shape[2]
    if not 1 <= m <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {m}")
    _need(min(layers, T, Hkv, Lmax, d) >= 1, "the caches must not be empty")
    _need(vc.shape == kc.shape, "k_cache and v_cache must have one shape")
    _need(kd.shape == (layers, T, m, Hkv, d) and vd.shape == kd.shape,
          f"drafts must be [{layers}, {T}, m, {Hkv}, {d}]")
    strides = []
    for x in (kc, vc, kd, vd):
        st = x.stride()
        if x.dtype is not kc.dtype or x.element_size() != 2 or (st[4] != 1 and d > 1):
            raise ValueError("caches and drafts must share one 16-bit dtype and be contiguous along the head dim")
        strides += st[:4]
    i32 = t.int32
    for x, shape, n in ((tokens, (T, m), "tokens"), (target, (T, m), "target"), (lens, (T,), "lens"),
                        (next_pos, (T,), "next_pos")):
        _plain(x, shape, i32, n)
    shared = parents.dim() == 1
    _plain(parents, (m,) if shared else (T, m), i32, "parents")
    lead = tuple(kc.shape[:3]) if k_cache.dim() == 5 else (T, Hkv)
    _need((scores is None) == (draft_scores is None), "scores and draft_scores go together")
    for x, last, dtype, n in ((scores, Lmax, t.float32, "scores"), (draft_scores, m, t.float32, "draft_scores"),
                              (positions, Lmax, i32, "positions")):
        if x is not None:
            _on_device(t, dev, **{n: x})
            _plain(x, lead + (last,), dtype, n)
    if dev_err is not None:
        _on_device(t, dev, dev_err=dev_err)
    ints = t.empty((m + 4) * T, dtype=i32, device=dev)  # one allocation for the five results
    r = Accepted(ints[4 * T:].view(T, m), ints[:T], ints[T:2 * T], ints[2 * T:3 * T], ints[3 * T:4 * T])
    with t.cuda.device(dev):
        rc = lib().mb_tree_accept(tokens.data_ptr(), parents.data_ptr(), 1 if shared else 0, target.data_ptr(),
                                  lens.data_ptr(), next_pos.data_ptr(), kc.data_ptr(), vc.data_ptr(), kd.data_ptr(),
                                  vd.data_ptr(), _Strides16(*strides), layers, T, m, Hkv, Lmax, d,
                                  None if scores is None else scores.data_ptr(),
                                  None if scores is None else draft_scores.data_ptr(),
                                  None if positions is None else positions.data_ptr(), r.path.data_ptr(),
                                  r.counts.data_ptr(), r.next_ids.data_ptr(), r.lens.data_ptr(), r.next_pos.data_ptr(),
                                  None if dev_err is None else dev_err.data_ptr(), stream_of(dev))
    if rc != 0:
        check(rc, "mb_tree_accept")
    return r


__all__ = ["Accepted", "MAX_NODES", "accept_tree", "tree_attention", "tree_depths", "tree_masks"]
