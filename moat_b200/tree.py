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


def _device_index(x, name: str) -> int:
    """Index of the CUDA device a tensor lies on."""
    try:
        idx = x.get_device()
    except AttributeError:
        raise TypeError(f"{name} must be a torch CUDA tensor") from None
    if idx < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return idx


def _on_device(idx: int, names, tensors) -> None:
    for name, x in zip(names, tensors):
        if _device_index(x, name) != idx:
            raise ValueError(f"{name} must be on cuda:{idx}")


def _plain(x, shape, dtype, name) -> None:
    """A contiguous tensor of one shape and dtype."""
    if x.dtype is not dtype or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)}")


def _strides(tensors, axes: int, dtype, what: str):
    """The leading strides of tensors of one dtype that are contiguous along their last axis."""
    out = ()
    for x in tensors:
        st = x.stride()
        if x.dtype is not dtype or (st[axes] != 1 and x.shape[axes] > 1):
            raise ValueError(what)
        out += st[:axes]
    return out


class _Workspaces:
    """Scratch per (device, stream), grown as needed; the kernels expect no initial contents,
    and calls that share a buffer are ordered by their stream. A buffer that was outgrown is
    kept: a captured graph may still use it."""

    def __init__(self):
        self._bufs, self._outgrown = {}, []

    def get(self, t, idx: int, stream: int, nbytes: int):
        buf = self._bufs.get((idx, stream))
        if buf is None or buf.numel() < nbytes:
            if buf is not None:
                self._outgrown.append(buf)
                nbytes = max(nbytes, 2 * buf.numel())
            buf = t.empty(max(nbytes, 1 << 20), dtype=t.uint8, device=t.device("cuda", idx))
            self._bufs[(idx, stream)] = buf
        return buf


def _on(t, idx: int, call):
    """``call(stream)`` with device ``idx`` current."""
    if idx == t.cuda.current_device():
        return call(stream_of(idx))
    with t.cuda.device(idx):
        return call(stream_of(idx))


_Strides18 = ctypes.c_int64 * 18
_Strides16 = ctypes.c_int64 * 16
_ws = _Workspaces()
_sizes = {}  # workspace bytes by geometry
_ATTN_NAMES = ("q", "k_cache", "v_cache", "lens", "k_draft", "v_draft", "masks")


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

    Scratch belongs to the stream; a captured graph keeps that of the stream it was captured
    on, so its replays and other calls of that stream must not overlap.

    fp32 scores, softmax and sums; one rounding at the output (and one of each unnormalised
    probability to the inputs' type before its product with V). Repeated calls give the same
    bits. Returns ``out``, or ``(out, scores_out, draft_scores)`` with ``scores``.
    """
    t = _lib.torch()
    idx = _device_index(q, "q")
    _on_device(idx, _ATTN_NAMES, (q, k_cache, v_cache, lens, k_draft, v_draft, masks))
    if q.dim() != 4 or k_cache.dim() != 4:
        raise ValueError("q must be [T, m, H, d] and the caches [T, Hkv, Lmax, d]")
    T, m, H, d = q.shape
    cache = k_cache.shape
    Hkv, Lmax = cache[1], cache[2]
    if not 1 <= m <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {m}")
    if T < 1 or Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"{H} query heads do not divide among {Hkv} KV heads")
    if not 1 <= d <= 256:
        raise ValueError(f"head dim must be 1 to 256, got {d}")
    if cache != (T, Hkv, Lmax, d) or v_cache.shape != cache:
        raise ValueError(f"k_cache / v_cache must be [{T}, {Hkv}, Lmax, {d}]")
    drafts = (T, m, Hkv, d)
    if k_draft.shape != drafts or v_draft.shape != drafts:
        raise ValueError(f"k_draft / v_draft must be {list(drafts)}")
    dt = q.dtype
    if dt is not t.float16 and dt is not t.bfloat16:
        raise ValueError("q must be fp16 or bf16")
    _plain(lens, (T,), t.int32, "lens")
    shared = masks.dim() == 1
    _plain(masks, (m,) if shared else (T, m), t.int64, "masks")
    if out is None:
        out = t.empty((T, m, H, d), dtype=dt, device=q.device)
    elif _device_index(out, "out") != idx or out.shape != q.shape:
        raise ValueError(f"out must be [{T}, {m}, {H}, {d}] on cuda:{idx}")
    strides = _strides((q, k_cache, v_cache, k_draft, v_draft, out), 3, dt,
                       "q, out, caches and drafts must share one dtype and be contiguous along the head dim")
    sc = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not math.isfinite(sc):
        raise ValueError("scale must be finite")
    ps = pso = pds = None
    if scores is not None:
        scores_out = scores if scores_out is None else scores_out
        if draft_scores is None:
            draft_scores = t.empty((T, Hkv, m), dtype=t.float32, device=q.device)
        _on_device(idx, ("scores", "scores_out", "draft_scores"), (scores, scores_out, draft_scores))
        f32, rows = t.float32, (T, Hkv, Lmax)
        _plain(scores, rows, f32, "scores")
        _plain(scores_out, rows, f32, "scores_out")
        _plain(draft_scores, (T, Hkv, m), f32, "draft_scores")
        ps, pso, pds = scores.data_ptr(), scores_out.data_ptr(), draft_scores.data_ptr()
    elif scores_out is not None or draft_scores is not None:
        raise ValueError("scores_out and draft_scores need scores")
    if dev_err is not None:
        _on_device(idx, ("dev_err",), (dev_err,))
    L = lib()
    geometry = (T, m, H, Hkv, Lmax, d, ps is not None)
    nbytes = _sizes.get(geometry)
    if nbytes is None:
        nbytes = _sizes[geometry] = int(L.mb_tree_attn_workspace_size(*geometry))

    def call(st):
        ws = _ws.get(t, idx, st, nbytes)
        return L.mb_tree_attn(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr(),
                              k_draft.data_ptr(), v_draft.data_ptr(), masks.data_ptr(), shared, out.data_ptr(),
                              _Strides18(*strides), dt is t.bfloat16, T, m, H, Hkv, Lmax, d, sc, ps, pso, pds,
                              ws.data_ptr(), ws.numel(), None if dev_err is None else dev_err.data_ptr(), st)

    rc = _on(t, idx, call)
    if rc != 0:
        check(rc, "mb_tree_attn")
    return out if ps is None else (out, scores_out, draft_scores)


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


_ACCEPT_NAMES = ("tokens", "parents", "target", "lens", "next_pos", "v_cache", "k_draft", "v_draft")


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
    t = _lib.torch()
    idx = _device_index(k_cache, "k_cache")
    _on_device(idx, _ACCEPT_NAMES, (tokens, parents, target, lens, next_pos, v_cache, k_draft, v_draft))
    kc, vc, kd, vd = (_five(x, n) for x, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (k_draft, "k_draft"),
                                               (v_draft, "v_draft")))
    layers, T, Hkv, Lmax, d = kc.shape
    drafts = kd.shape
    m = drafts[2]
    if not 1 <= m <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {m}")
    if min(layers, T, Hkv, Lmax, d) < 1:
        raise ValueError("the caches must not be empty")
    if vc.shape != kc.shape:
        raise ValueError("k_cache and v_cache must have one shape")
    if drafts != (layers, T, m, Hkv, d) or vd.shape != drafts:
        raise ValueError(f"drafts must be [{layers}, {T}, m, {Hkv}, {d}]")
    what = "caches and drafts must share one 16-bit dtype and be contiguous along the head dim"
    if kc.element_size() != 2:
        raise ValueError(what)
    strides = _strides((kc, vc, kd, vd), 4, kc.dtype, what)
    i32 = t.int32
    _plain(tokens, (T, m), i32, "tokens")
    _plain(target, (T, m), i32, "target")
    _plain(lens, (T,), i32, "lens")
    _plain(next_pos, (T,), i32, "next_pos")
    shared = parents.dim() == 1
    _plain(parents, (m,) if shared else (T, m), i32, "parents")
    if (scores is None) != (draft_scores is None):
        raise ValueError("scores and draft_scores go together")
    lead = (layers, T, Hkv) if k_cache.dim() == 5 else (T, Hkv)
    ps = pd = pp = None
    if scores is not None:
        _on_device(idx, ("scores", "draft_scores"), (scores, draft_scores))
        _plain(scores, lead + (Lmax,), t.float32, "scores")
        _plain(draft_scores, lead + (m,), t.float32, "draft_scores")
        ps, pd = scores.data_ptr(), draft_scores.data_ptr()
    if positions is not None:
        _on_device(idx, ("positions",), (positions,))
        _plain(positions, lead + (Lmax,), i32, "positions")
        pp = positions.data_ptr()
    if dev_err is not None:
        _on_device(idx, ("dev_err",), (dev_err,))
    ints = t.empty((m + 4) * T, dtype=i32, device=kc.device)  # one allocation for the five results
    path, counts, next_ids, new_lens, new_pos = ints.split_with_sizes([T * m, T, T, T, T])
    p0 = ints.data_ptr()
    p1, step = p0 + 4 * T * m, 4 * T
    rc = _on(t, idx, lambda st: lib().mb_tree_accept(
        tokens.data_ptr(), parents.data_ptr(), shared, target.data_ptr(), lens.data_ptr(), next_pos.data_ptr(),
        kc.data_ptr(), vc.data_ptr(), kd.data_ptr(), vd.data_ptr(), _Strides16(*strides), layers, T, m, Hkv, Lmax, d,
        ps, pd, pp, p0, p1, p1 + step, p1 + 2 * step, p1 + 3 * step, None if dev_err is None else dev_err.data_ptr(),
        st))
    if rc != 0:
        check(rc, "mb_tree_accept")
    return Accepted(path.view(T, m), counts, next_ids, new_lens, new_pos)


__all__ = ["Accepted", "MAX_NODES", "accept_tree", "tree_attention", "tree_depths", "tree_masks"]
