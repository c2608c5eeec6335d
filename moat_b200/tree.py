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

from typing import NamedTuple

import numpy as np

from . import _lib
from ._lib import check

MAX_NODES = 64  # one bit per node in a mask

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


# ---------------------------------------------------------------------------
# Arguments. The binding (csrc/bind.cpp) tests all of a call's tensors; only where one does
# not fit does a second, slower pass here find out which and say so.
# ---------------------------------------------------------------------------
def _device_index(x, name: str) -> int:
    """Index of the CUDA device a tensor lies on."""
    try:
        idx = x.get_device()
    except AttributeError:
        raise TypeError(f"{name} must be a torch CUDA tensor") from None
    if idx < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return idx


def _on_device(idx: int, **tensors) -> None:
    for name, x in tensors.items():
        if x is not None and _device_index(x, name) != idx:
            raise ValueError(f"{name} must be on cuda:{idx}")


def _plain(x, shape, dtype, name) -> None:
    """A contiguous tensor of one shape and dtype."""
    if x.dtype is not dtype or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)}")


def _error_word(t, x) -> None:
    """The device error word, if there is one."""
    if x is not None and (x.dtype is not t.int32 or x.numel() < 1):
        raise ValueError("dev_err must be an int32 tensor of one word or more")


def _rows(dtype, what: str, *tensors) -> None:
    """Tensors of one dtype, contiguous along their last axis."""
    for x in tensors:
        if x.dtype is not dtype or (x.stride(-1) != 1 and x.shape[-1] > 1):
            raise ValueError(what)


def _own_places(**tensors) -> None:
    """Tensors that are written: no broadcast axes."""
    for name, x in tensors.items():
        if any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
            raise ValueError(f"{name} is written and must not be broadcast along an axis")


_modules = []


def _torch():
    if not _modules:
        _modules.append(_lib.torch())
    return _modules[0]


def _done(result, entry: str, explain, *args):
    """The result of a call through the binding: a status is an error, None means that an
    argument does not fit, which ``explain(*args)`` says."""
    if result is None:
        explain(*args)
        raise ValueError(f"arguments of {entry} do not fit")
    if type(result) is int:
        check(result, entry)
    return result


def _check_attention(q, k_cache, v_cache, lens, k_draft, v_draft, masks, out, scores, scores_out, draft_scores, dev_err):
    t = _torch()
    given, out = out, q if out is None else out
    if scores is not None:
        scores_out = scores if scores_out is None else scores_out
    idx = _device_index(q, "q")
    _on_device(idx, k_cache=k_cache, v_cache=v_cache, lens=lens, k_draft=k_draft, v_draft=v_draft, masks=masks, out=out,
               scores=scores, scores_out=scores_out, draft_scores=draft_scores, dev_err=dev_err)
    if q.dim() != 4 or k_cache.dim() != 4:
        raise ValueError("q must be [T, m, H, d] and the caches [T, Hkv, Lmax, d]")
    T, m, H, d = q.shape
    Hkv, Lmax = k_cache.shape[1:3]
    if not 1 <= m <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {m}")
    if T < 1 or Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"{H} query heads do not divide among {Hkv} KV heads")
    if not 1 <= d <= 256:
        raise ValueError(f"head dim must be 1 to 256, got {d}")
    if k_cache.shape != (T, Hkv, Lmax, d) or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache / v_cache must be [{T}, {Hkv}, Lmax, {d}]")
    if k_draft.shape != (T, m, Hkv, d) or v_draft.shape != k_draft.shape:
        raise ValueError(f"k_draft / v_draft must be [{T}, {m}, {Hkv}, {d}]")
    if q.dtype not in (t.float16, t.bfloat16):
        raise ValueError("q must be fp16 or bf16")
    _plain(lens, (T,), t.int32, "lens")
    _plain(masks, (m,) if masks.dim() == 1 else (T, m), t.int64, "masks")
    if out.shape != q.shape:
        raise ValueError(f"out must be [{T}, {m}, {H}, {d}]")
    _rows(q.dtype, "q, out, caches and drafts must share one dtype and be contiguous along the head dim", q, k_cache,
          v_cache, k_draft, v_draft, out)
    _own_places(out=out)
    if scores is not None:
        if given is not None and out.data_ptr() == q.data_ptr():
            raise ValueError("with scores, out must not be q")
        _plain(scores, (T, Hkv, Lmax), t.float32, "scores")
        _plain(scores_out, (T, Hkv, Lmax), t.float32, "scores_out")
        if draft_scores is not None:
            _plain(draft_scores, (T, Hkv, m), t.float32, "draft_scores")
    elif scores_out is not None or draft_scores is not None:
        raise ValueError("scores_out and draft_scores need scores")
    _error_word(t, dev_err)


def tree_attention(q, k_cache, v_cache, lens, k_draft, v_draft, masks, *, scale=None, out=None, scores=None,
                   scores_out=None, draft_scores=None, dev_err=None):
    """Attention of every node of every trace's tree.

    * ``q [T, m, H, d]``, ``k_cache`` / ``v_cache [T, Hkv, Lmax, d]`` (the first ``lens[t]``
      rows valid), ``k_draft`` / ``v_draft [T, m, Hkv, d]``: fp16 or bf16, CUDA, the last
      axis contiguous, other strides free; ``d <= 256``.
    * ``lens`` int32 ``[T]``, ``masks`` int64 ``[T, m]`` or ``[m]`` (one tree for every
      trace): node ``i`` sees all committed rows and the nodes whose bit is set. A mask of 0
      marks padding: the node sees nothing and its output is 0.
    * ``out``: optional result ``[T, m, H, d]`` that overlaps no input (without ``scores`` it
      may be ``q`` itself); ``scale`` defaults to ``1/sqrt(d)``.
    * ``scores`` float32 ``[T, Hkv, Lmax]``: also compute, for every row, its attention
      weight summed over the nodes and the heads of its group. ``scores_out`` (default: in
      place) gets ``scores`` plus that sum in the first ``lens[t]`` rows and keeps the
      others; ``draft_scores`` float32 ``[T, Hkv, m]`` gets the sums of the draft's rows.
    * ``dev_err``: optional int32 CUDA tensor whose first word receives device error bits
      (bounded waits).

    Scratch comes from torch's allocator for the length of the call (a captured call's from
    its graph's pool); with scores and up to 16 rows (nodes x heads of a group) it holds a
    float per row and cached row.

    fp32 scores, softmax and sums; one rounding at the output (and one of each unnormalised
    probability to the inputs' type before its product with V). Values that are not finite
    reach only the nodes that see their row. Repeated calls give the same bits. Returns ``out``,
    or ``(out, scores_out, draft_scores)`` with ``scores``.
    """
    r = _lib.bind().attention(q, k_cache, v_cache, lens, k_draft, v_draft, masks, scale, out, scores, scores_out,
                              draft_scores, dev_err)
    if r is None or type(r) is int:
        _done(r, "mb_tree_attn", _check_attention, q, k_cache, v_cache, lens, k_draft, v_draft, masks, out, scores,
              scores_out, draft_scores, dev_err)
    return r


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


def _check_accept(tokens, parents, target, lens, next_pos, k_cache, v_cache, k_draft, v_draft, scores, draft_scores,
                  positions, dev_err):
    t = _torch()
    idx = _device_index(k_cache, "k_cache")
    _on_device(idx, tokens=tokens, parents=parents, target=target, lens=lens, next_pos=next_pos, v_cache=v_cache,
               k_draft=k_draft, v_draft=v_draft, scores=scores, draft_scores=draft_scores, positions=positions,
               dev_err=dev_err)
    kc, vc, kd, vd = (_five(x, n) for x, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (k_draft, "k_draft"),
                                               (v_draft, "v_draft")))
    layers, T, Hkv, Lmax, d = kc.shape
    m = kd.shape[2]
    if not 1 <= m <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {m}")
    if min(layers, T, Hkv, Lmax, d) < 1:
        raise ValueError("the caches must not be empty")
    if vc.shape != kc.shape:
        raise ValueError("k_cache and v_cache must have one shape")
    if kd.shape != (layers, T, m, Hkv, d) or vd.shape != kd.shape:
        raise ValueError(f"drafts must be [{layers}, {T}, m, {Hkv}, {d}]")
    what = "caches and drafts must share one 16-bit dtype and be contiguous along the head dim"
    if kc.element_size() != 2:
        raise ValueError(what)
    _rows(kc.dtype, what, kc, vc, kd, vd)
    _own_places(k_cache=kc, v_cache=vc)
    i32 = t.int32
    for x, shape, name in ((tokens, (T, m), "tokens"), (target, (T, m), "target"), (lens, (T,), "lens"),
                           (next_pos, (T,), "next_pos"), (parents, (m,) if parents.dim() == 1 else (T, m), "parents")):
        _plain(x, shape, i32, name)
    if (scores is None) != (draft_scores is None):
        raise ValueError("scores and draft_scores go together")
    lead = k_cache.shape[:-2]
    if scores is not None:
        _plain(scores, (*lead, Lmax), t.float32, "scores")
        _plain(draft_scores, (*lead, m), t.float32, "draft_scores")
    if positions is not None:
        _plain(positions, (*lead, Lmax), i32, "positions")
    _error_word(t, dev_err)


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
    r = _lib.bind().accept(tokens, parents, target, lens, next_pos, k_cache, v_cache, k_draft, v_draft, scores,
                           draft_scores, positions, dev_err)
    if r is None or type(r) is int:
        _done(r, "mb_tree_accept", _check_accept, tokens, parents, target, lens, next_pos, k_cache, v_cache, k_draft,
              v_draft, scores, draft_scores, positions, dev_err)
    return Accepted._make(r)


__all__ = ["Accepted", "MAX_NODES", "accept_tree", "tree_attention", "tree_depths", "tree_masks"]
