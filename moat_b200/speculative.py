"""Drafted decoding with an ``Int4Decoder``'s weights: several tokens per step and trace,
in a cache of fixed size.

A step runs a tree of drafted tokens through the model at once: the INT4 GEMMs see
``N * m`` rows (they stream the weights once per 32 rows either way), ``tree_attention``
lets every node see the trace's cache and its own ancestors, ``accept_tree`` keeps the path
that the model itself would have chosen and appends its keys and values to the caches of
all layers. The tokens are those of greedy decoding with exact softmax attention (the
reference's PyTorch decoder, ``transformer.py:110-119``); ``Int4Decoder.step`` uses the exp
table's softmax, whose attention differs by about 3e-4, so near-ties may fall the other way.

With a ``budget`` the caches hold at most that many rows (plus those since the last
eviction): ``tree_attention`` sums up the attention weight of every cached row and
``evict_cache`` keeps the recent rows, the first ones and the heaviest. What was drafted has a
say in which: every drafted node counts, also one that is rejected afterwards; a missing one
(-1), and what hangs on it, does not.

    dec = Int4Decoder(cfg, n_traces=16)
    spec = TreeDecoder(dec, parents=[-1, 0, 1, 2, 0], budget=512, capacity=640)
    spec.prefill(prompt_ids)
    tokens = spec.generate(steps=100, draft=lookup_draft)
"""

from __future__ import annotations

import numpy as np

from . import _lib
from ._lib import check, check_device, lib, stream_of
from .decode import rope_table
from .evict import evict_cache
from .tree import MAX_NODES, accept_tree, tree_attention, tree_depths, tree_masks


def lookup_draft(history, m: int):
    """``m - 1`` drafted tokens of a chain by lookup: what followed the latest earlier
    occurrence of the history's last two tokens (else of its last one); -1, which is never
    accepted, where nothing is found. ``history``: list of token ids, newest last."""
    for n in (2, 1):
        key = history[-n:]
        for at in range(len(history) - n - 1, -1, -1):
            if history[at:at + n] == key:
                found = history[at + n:at + n + m - 1]
                return found + [-1] * (m - 1 - len(found))
    return [-1] * (m - 1)


class _Shape:
    """Device tables and activations of trees of one shape."""

    def __init__(self, dec, parents, device):
        t = _lib.torch()
        par = np.asarray(parents, dtype=np.int32)
        self.m = m = len(par)
        self.parents = t.from_numpy(par).to(device)
        self.masks = t.from_numpy(tree_masks(par)).to(device)
        self.depths = t.from_numpy(tree_depths(par)).to(device)
        self.nodes = t.arange(m, dtype=t.int64, device=device)
        cfg, N = dec.cfg, dec.N
        D, H, dh, F = cfg.hidden, cfg.heads, cfg.head_dim, cfg.ffn
        rows = N * m

        def f16(*shape):
            return t.empty(shape, dtype=t.float16, device=device)

        self.tokens = t.full((N, m), -1, dtype=t.int32, device=device)
        self.x = t.empty((rows, D), dtype=t.float32, device=device)
        self.h, self.o, self.att = f16(rows, D), f16(rows, D), f16(N, m, H, dh)
        self.q, self.gu, self.a = f16(N, m, H, dh), f16(rows, 2 * F), f16(rows, F)
        # every layer's projection is kept: its values are the draft's value rows
        self.qkv = f16(cfg.layers, N, m, 3 * D)
        self.k_draft = f16(cfg.layers, N, m, H, dh)
        self.v_draft = self.qkv[..., 2 * D:].view(cfg.layers, N, m, H, dh)
        self.draft_scores = t.zeros((cfg.layers, N, H, m), dtype=t.float32, device=device)


class TreeDecoder:
    """Drafted greedy decoding of a one-GPU ``Int4Decoder``'s traces.

    * ``parents``: the tree's shape, the same for every step (``parents[0] = -1``).
    * ``capacity``: rows of the caches (default: the decoder's ``max_len``);
      ``max_positions``: the longest sequence (default: ``capacity``, or eight times it
      with a budget).
    * ``budget``, ``recent``, ``sinks``: see ``evict_cache``; without a budget nothing is
      evicted, and no scores are kept.

    The caches are this object's own; traces may differ in length (``lens``, on the device).
    ``dev_err`` collects the device error bits; ``generate`` raises for them.
    """

    def __init__(self, dec, parents, capacity=None, budget=None, recent: int = 64, sinks: int = 4,
                 max_positions=None):
        t = _lib.require_cuda()
        if dec.world != 1:
            raise ValueError("drafted decoding runs on one GPU (world = 1)")
        cfg = dec.cfg
        self.dec, self.dev, self.N = dec, dec.dev, dec.N
        self.capacity = int(cfg.max_len if capacity is None else capacity)
        self.budget, self.recent, self.sinks = budget, int(recent), int(sinks)
        parents = list(parents)
        if not 1 <= len(parents) <= MAX_NODES:
            raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {len(parents)}")
        if budget is not None and not (self.recent + self.sinks <= budget <= self.capacity - len(parents)):
            raise ValueError("budget must hold the recent rows and the sinks and leave room for a tree")
        if max_positions is None:
            max_positions = self.capacity * (1 if budget is None else 8)
        self.max_positions = int(max_positions)
        self.cs = rope_table(cfg.head_dim, self.max_positions, cfg.theta).to(self.dev)
        self.shape = _Shape(dec, parents, self.dev)
        self.m = self.shape.m
        full = (cfg.layers, self.N, cfg.heads, self.capacity)
        self.k_cache = t.zeros(full + (cfg.head_dim,), dtype=t.float16, device=self.dev)
        self.v_cache = t.zeros_like(self.k_cache)
        self.scores = self.positions = None
        if budget is not None:
            self.scores = t.zeros(full, dtype=t.float32, device=self.dev)
            self.positions = t.zeros(full, dtype=t.int32, device=self.dev)
        self.lens = t.zeros(self.N, dtype=t.int32, device=self.dev)
        self.next_pos = t.zeros_like(self.lens)
        self.ids = t.zeros_like(self.lens)  # each trace's last chosen token, not yet in the cache
        self.pending = False  # no token has been chosen yet
        self.dev_err = t.zeros(1, dtype=t.int32, device=self.dev)
        self.logits = t.empty((self.N * self.m, cfg.vocab), dtype=t.float16, device=self.dev)
        self._logits_lm = (self.logits if dec.lm_cols == cfg.vocab
                           else t.empty((self.N * self.m, dec.lm_cols), dtype=t.float16, device=self.dev))
        self.target = t.zeros((self.N, self.m), dtype=t.int32, device=self.dev)
        self.history = [[] for _ in range(self.N)]
        self.rows = 0  # no trace has more cached rows than this
        self.longest = 0  # or a later position

    # -------------------------------------------------------------------------
    def _drafted_masks(self, s: _Shape):
        """Masks ``[N, m]`` of the tree in ``s.tokens``: a missing node, and what hangs on it,
        is padding."""
        t = _lib.torch()
        missing = ((s.tokens < 0).long() << s.nodes).sum(dim=1, keepdim=True)  # a bit per node
        return t.where((s.masks & missing) == 0, s.masks, 0)

    def _layers(self, s: _Shape):
        """The tree in ``s.tokens`` through all layers: leaves the draft's keys, values and
        scores in ``s``, the residual in ``s.x`` and the last layer's output in ``s.o``."""
        dec, cfg, L = self.dec, self.dec.cfg, lib()
        N, m, D, H, dh, F = self.N, s.m, cfg.hidden, cfg.heads, cfg.head_dim, cfg.ffn
        rows = N * m
        st = stream_of(self.dev)
        err = self.dev_err.data_ptr()
        p = lambda x: x.data_ptr()  # noqa: E731
        # a missing draft (-1) is embedded as token 0: no node sees it
        ids, masks = s.tokens.clamp(min=0), self._drafted_masks(s)
        check(L.mb_embed(p(ids), rows, p(dec.embed), cfg.vocab, D, p(s.x), err, st), "mb_embed")
        y = None
        for li, lw in enumerate(dec.layers):
            check(L.mb_add_rmsnorm(p(s.x), y, p(lw["attn_norm"]), rows, D, cfg.eps, p(s.h), st), "mb_add_rmsnorm")
            check(L.mb_int4_gemm(p(s.h), p(lw["wqkv"]), p(s.qkv[li]), rows, D, 3 * D, err, st), "qkv")
            check(L.mb_tree_rope(p(s.qkv[li]), 0, N, m, H, H, dh, p(self.next_pos), p(s.depths), 1, p(self.cs),
                                 self.max_positions, p(s.q), p(s.k_draft[li]), err, st), "mb_tree_rope")
            scores = {}
            if self.scores is not None:
                scores = dict(scores=self.scores[li], draft_scores=s.draft_scores[li])
            tree_attention(s.q, self.k_cache[li], self.v_cache[li], self.lens, s.k_draft[li], s.v_draft[li], masks,
                           scale=dec.scale, out=s.att, dev_err=self.dev_err, **scores)
            check(L.mb_int4_gemm(p(s.att), p(lw["wo"]), p(s.o), rows, D, D, err, st), "o_proj")
            check(L.mb_add_rmsnorm(p(s.x), p(s.o), p(lw["ffn_norm"]), rows, D, cfg.eps, p(s.h), st), "mb_add_rmsnorm")
            check(L.mb_int4_gemm(p(s.h), p(lw["wgu"]), p(s.gu), rows, D, 2 * F, err, st), "gate_up")
            check(L.mb_swiglu(p(s.gu), rows, F, p(s.a), st), "mb_swiglu")
            check(L.mb_int4_gemm(p(s.a), p(lw["wd"]), p(s.o), rows, F, D, err, st), "down")
            y = p(s.o)

    def _choose(self, s: _Shape):
        """The model's greedy choice at every node, into ``self.target``."""
        dec, cfg, L = self.dec, self.dec.cfg, lib()
        rows, st, err = self.N * s.m, stream_of(self.dev), self.dev_err.data_ptr()
        p = lambda x: x.data_ptr()  # noqa: E731
        check(L.mb_add_rmsnorm(p(s.x), p(s.o), p(dec.final_norm), rows, cfg.hidden, cfg.eps, p(s.h), st),
              "mb_add_rmsnorm")
        check(L.mb_int4_gemm(p(s.h), p(dec.lm_head), p(self._logits_lm), rows, cfg.hidden, dec.lm_cols, err, st),
              "lm_head")
        if self._logits_lm is not self.logits:
            self.logits.copy_(self._logits_lm[:, :cfg.vocab])
        check(L.mb_argmax_f16(p(self.logits), rows, cfg.vocab, p(self.target), st), "mb_argmax_f16")

    def _accept(self, s: _Shape, target):
        r = accept_tree(s.tokens, s.parents, target, self.lens, self.next_pos, self.k_cache, self.v_cache, s.k_draft,
                        s.v_draft, scores=self.scores,
                        draft_scores=None if self.scores is None else s.draft_scores, positions=self.positions,
                        dev_err=self.dev_err)
        self.lens.copy_(r.lens)
        self.next_pos.copy_(r.next_pos)
        self.ids.copy_(r.next_ids)
        return r

    def _read_lengths(self):
        """The true lengths in place of the bounds; waits for the device."""
        self.rows, self.longest = int(self.lens.max()), int(self.next_pos.max())

    def _make_room(self, m: int):
        """Room for m more rows in every trace; evicts where there is none. The lengths stay on
        the device: they are read only where the bounds kept here leave no room."""
        if self.rows + m > self.capacity or self.longest + m > self.max_positions:
            self._read_lengths()
        if self.longest + m > self.max_positions:
            raise ValueError("the sequence is longer than max_positions")
        if self.rows + m > self.capacity:
            if self.budget is None or self.budget + m > self.capacity:
                raise ValueError("KV cache is full")
            _, _, lens = evict_cache(self.k_cache, self.v_cache, self.scores, self.positions, self.lens, self.next_pos,
                                     self.budget, recent=self.recent, sinks=self.sinks)
            self.lens.copy_(lens)
            self.rows = min(self.rows, self.budget)
        self.rows += m
        self.longest += m

    # -------------------------------------------------------------------------
    def prefill(self, prompt_ids, chunk: int = 32):
        """Run a prompt ``[N, P]`` through the model, ``chunk`` positions at a time as a chain
        whose every node is accepted. All but the last token end up in the caches; the last
        one is the next step's root. After tokens or another prompt, the token chosen last, which
        is not in the caches yet, comes before this one. Beside a budget that leaves less room
        than a chunk, chunks are smaller. A prompt that does not fit is refused before anything
        changes."""
        t = _lib.torch()
        if prompt_ids.dim() != 2 or prompt_ids.shape[0] != self.N or prompt_ids.shape[1] < 1:
            raise ValueError(f"prompt ids must be [{self.N}, P]")
        if not 1 <= chunk <= MAX_NODES:
            raise ValueError(f"chunk must be 1 to {MAX_NODES}")
        ids = prompt_ids.to(device=self.dev, dtype=t.int32)
        row_tokens = ids.tolist()
        if self.pending:
            ids = t.cat([self.ids.unsqueeze(1), ids], 1)
        P, at, s = int(ids.shape[1]), 0, None
        self._read_lengths()
        if self.longest + P - 1 > self.max_positions:
            raise ValueError("the sequence is longer than max_positions")
        if self.budget is None and self.rows + P - 1 > self.capacity:
            raise ValueError("KV cache is full")
        self.ids.copy_(ids[:, 0])
        self.pending = True
        while at < P - 1:
            n = min(chunk, P - 1 - at)
            if self.budget is not None:
                n = min(n, self.capacity - min(self.rows, self.budget))
            if s is None or s.m != n:
                s = _Shape(self.dec, range(-1, n - 1), self.dev)
            self._make_room(n)
            s.tokens.copy_(ids[:, at:at + n])
            s.tokens[:, 0].copy_(self.ids)  # an idle trace stays idle
            self._layers(s)
            self._accept(s, ids[:, at + 1:at + n + 1].contiguous())
            at += n
        for hist, row in zip(self.history, row_tokens):
            hist.extend(row)

    def step(self, drafts):
        """Verify one tree per trace: ``drafts`` int32 ``[N, m - 1]`` (nodes 1 to m - 1; -1
        where there is none), host or device. Returns the device ``Accepted``; the new
        tokens of trace n are the accepted drafts in ``path`` and ``next_ids[n]``."""
        t = _lib.torch()
        s = self.shape
        drafts = t.as_tensor(drafts, dtype=t.int32)
        if tuple(drafts.shape) != (self.N, self.m - 1):
            raise ValueError(f"drafts must be [{self.N}, {self.m - 1}]")
        self._make_room(self.m)
        self.pending = True
        s.tokens[:, 0].copy_(self.ids)
        s.tokens[:, 1:].copy_(drafts)
        self._layers(s)
        self._choose(s)
        return self._accept(s, self.target)

    def generate(self, steps: int, draft=lookup_draft):
        """``steps`` verified steps; ``draft(history, m)`` gives a trace's ``m - 1`` tokens.
        Returns the new tokens of every trace (lists of different lengths)."""
        first = [len(hist) for hist in self.history]
        for _ in range(steps):
            drafts = [draft(hist, self.m) for hist in self.history]
            r = self.step(drafts)
            path, nxt = r.path.tolist(), r.next_ids.tolist()  # also waits for the step
            check_device(int(self.dev_err), "drafted decoding")
            for hist, d, nodes, token in zip(self.history, drafts, path, nxt):
                hist.extend(d[i - 1] for i in nodes[1:] if i > 0)
                if token >= 0:
                    hist.append(token)
            self._read_lengths()
        return [hist[n:] for hist, n in zip(self.history, first)]


__all__ = ["TreeDecoder", "lookup_draft"]
