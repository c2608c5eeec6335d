"""TreeDecoder over several calls: missing drafts, budgets, bounds, prompts after prompts.

The oracle is the fp32 decoder on the host; under a budget it sees, per layer and head, the rows
that the caches held. Logits agree as in test_gpu_speculative.py (2e-2), and so do the weights
that the rows have drawn. A row that was evicted drew no more than one that stayed, up to twice
that tolerance.
"""

import numpy as np
import pytest

from test_gpu_speculative import make, prompt, run_checked

pytestmark = pytest.mark.gpu

TOL = 2e-2


class Oracle:
    """One trace's rows, per layer and head, with the weight that each has drawn."""

    def __init__(self, dec, rows):
        import torch
        self.t, self.w, self.cfg = torch, dec.dense_weights(), dec.cfg
        H, dh, layers = self.cfg.heads, self.cfg.head_dim, len(self.w["layers"])
        self.k, self.v = (torch.zeros(layers, H, rows, dh) for _ in range(2))
        self.drawn = np.zeros((layers, H, rows))

    def token(self, tok, pos, first, cached):
        """Logits after a token at position pos of a chain that begins at first, over the positions
        cached[layer][head]."""
        t, w, cfg = self.t, self.w, self.cfg
        H, dh = cfg.heads, cfg.head_dim
        norm = lambda x, g: x * t.rsqrt(x.pow(2).mean() + cfg.eps) * g  # noqa: E731
        x = w["embed"][tok].float()
        for li, lw in enumerate(w["layers"]):
            qkv = (norm(x, lw["attn_norm"]) @ lw["wqkv"]).view(3, H, dh)
            q, k = (t.view_as_real(t.view_as_complex(y.reshape(H, dh // 2, 2).contiguous()) * w["cis"][pos]).reshape(H, dh)
                    for y in qkv[:2])
            self.k[li, :, pos], self.v[li, :, pos] = k, qkv[2]
            att = []
            for h in range(H):
                rows = sorted(cached[li][h]) + list(range(first, pos + 1))
                p = t.softmax(self.k[li, h, rows] @ q[h] / dh ** 0.5, 0)
                self.drawn[li, h, rows] += p.numpy()
                att.append(p @ self.v[li, h, rows])
            x = x + t.cat(att) @ lw["wo"]
            g, u = (norm(x, lw["ffn_norm"]) @ lw["wgu"]).chunk(2)
            x = x + (t.nn.functional.silu(g) * u) @ lw["wd"]
        return (norm(x, w["final_norm"]) @ w["lm_head"]).numpy()


def cached_positions(spec, lens=None):
    """Of every trace, layer and head."""
    lens = spec.lens.tolist() if lens is None else lens
    pos = spec.positions.cpu().numpy()
    return [[[set(pos[li, n, h, :lens[n]].tolist()) for h in range(pos.shape[2])] for li in range(pos.shape[0])]
            for n in range(spec.N)]


def watch(spec, monkeypatch):
    """Records what happens to the caches: ("rows", first positions, cached, counts, logits) for every
    accepted chain and ("evict", before, after)."""
    from moat_b200 import speculative
    events = []
    accept, evict = spec._accept, speculative.evict_cache

    def spy_accept(s, target):
        first, cached = spec.next_pos.tolist(), cached_positions(spec)
        r = accept(s, target)
        assert all(p[:c] == list(range(c)) for p, c in zip(r.path.tolist(), r.counts.tolist()))  # chains
        logits = spec.logits.view(spec.N, spec.m, -1).float().cpu().numpy() if target is spec.target else None
        events.append(("rows", first, cached, r.counts.tolist(), logits))
        return r

    def spy_evict(*args, **kw):
        before = cached_positions(spec)
        r = evict(*args, **kw)
        events.append(("evict", before, cached_positions(spec, r[2].tolist()), spec.next_pos.tolist()))
        return r

    monkeypatch.setattr(spec, "_accept", spy_accept)
    monkeypatch.setattr(speculative, "evict_cache", spy_evict)
    return events


def check_events(dec, spec, events):
    """Replays every trace on the host; the number of evictions that took rows out."""
    evictions = 0
    for n, hist in enumerate(spec.history):
        o = Oracle(dec, len(hist))
        for what, first, cached, *rest in events:
            if what == "rows":
                for j in range(rest[0][n]):
                    want = o.token(hist[first[n] + j], first[n] + j, first[n], cached[n])
                    if rest[1] is not None:
                        np.testing.assert_allclose(rest[1][n, j], want, rtol=TOL, atol=TOL)
                        assert hist[first[n] + j + 1] == int(np.argmax(rest[1][n, j]))
                continue
            before, after, nxt = first[n], cached[n], rest[0][n]
            for li, heads in enumerate(before):
                for h, rows in enumerate(heads):
                    guarded = {p for p in rows if p >= nxt - spec.recent or p < spec.sinks}
                    gone, stayed = rows - after[li][h], after[li][h] - guarded
                    assert after[li][h] <= rows and guarded <= after[li][h]
                    assert len(after[li][h]) == min(len(rows), spec.budget)
                    evictions += bool(gone)
                    if gone and stayed:
                        most = max(o.drawn[li, h, p] for p in gone)
                        assert most <= min(o.drawn[li, h, p] for p in stayed) + 2 * TOL * (1 + most)
        pos, got = spec.positions[:, n].cpu().numpy(), spec.scores[:, n].cpu().numpy()
        for li in range(pos.shape[0]):
            for h in range(pos.shape[1]):
                rows = int(spec.lens[n])
                np.testing.assert_allclose(got[li, h, :rows], o.drawn[li, h, pos[li, h, :rows]], rtol=TOL, atol=TOL)
    assert int(spec.dev_err) == 0
    return evictions


@pytest.mark.parametrize("drafts,nodes", [([-1, -1, -1], 1), ([5, -1, 7], 3), ([-1, 5, 7], 2), ([5, 6, 7], 4)])
def test_only_drafted_nodes_weigh_the_rows(cuda, drafts, nodes):
    """Every real node gives each head a weight of 1 in all (here to 1e-3, the fp32 sums of 40
    rows); a missing one, and what hangs on it, none."""
    dec, spec = make(cuda, parents=[-1, 0, 0, 1], capacity=60, budget=50, recent=8)
    spec.prefill(prompt(cuda, 3, 30, 1000))
    n = spec.lens.tolist()[0]
    before = spec.scores[..., :n].double().sum(-1)
    spec.step(np.array([drafts] * 3, np.int32))
    added = spec.scores[..., :n].double().sum(-1) - before + spec.shape.draft_scores.double().sum(-1)
    assert bool(((added - nodes).abs() < 1e-3).all())


@pytest.mark.parametrize("parents", [[-1], [-1, 0, 1, 2]])
def test_a_long_run_without_drafts(cuda, monkeypatch, parents):
    """Missing drafts draw nothing: the rows that stay are those that the tokens themselves weigh most."""
    dec, spec = make(cuda, parents=parents, capacity=56, budget=40, recent=12, sinks=2, max_positions=400)
    events = watch(spec, monkeypatch)
    spec.prefill(prompt(cuda, 3, 60, 1000), chunk=8)
    spec.generate(30, lambda hist, m: [-1] * (m - 1))
    assert spec.next_pos.tolist() == [89] * 3
    assert check_events(dec, spec, events) >= 3 * 4 * 3  # traces, heads of all layers, times


@pytest.mark.parametrize("kw", [dict(capacity=24), dict(capacity=40, max_positions=24)])
def test_steps_fill_the_cache(cuda, kw):
    """Rejected drafts take no room, in calls of step() as in generate()."""
    dec, spec = make(cuda, parents=[-1, 0, 1, 2, 3], **kw)
    spec.prefill(prompt(cuda, 3, 5, 1000))
    none = np.full((3, 4), -1, np.int32)
    for i in range(16):
        assert spec.lens.tolist() == [4 + i] * 3
        spec.step(none)
    with pytest.raises(ValueError):
        spec.step(none)
    assert spec.lens.tolist() == [20] * 3


def test_step_and_generate_keep_the_same_rows(cuda):
    runs = []
    for stepwise in (True, False):
        dec, spec = make(cuda, parents=[-1, 0, 1, 0], capacity=56, budget=40, recent=12, sinks=2, max_positions=400)
        spec.prefill(prompt(cuda, 3, 30, 1000), chunk=8)
        if stepwise:
            for _ in range(60):
                spec.step(np.full((3, 3), -1, np.int32))
        else:
            spec.generate(60, lambda hist, m: [-1] * 3)
        runs.append((spec.ids.tolist(), spec.lens.tolist(), spec.positions.tolist(), spec.scores.tolist()))
    assert runs[0] == runs[1]


@pytest.mark.parametrize("parents,capacity", [([-1, 0, 1, 2], 46), ([-1], 41)])
def test_a_prompt_in_little_room(cuda, monkeypatch, parents, capacity):
    """Room for fewer rows than a chunk beside the budget: the chunks become smaller."""
    dec, spec = make(cuda, parents=parents, capacity=capacity, budget=40, recent=12, sinks=2, max_positions=400)
    events = watch(spec, monkeypatch)
    spec.prefill(prompt(cuda, 3, 60, 1000))
    assert spec.next_pos.tolist() == [59] * 3
    spec.generate(5, lambda hist, m: [-1] * (m - 1))
    assert spec.next_pos.tolist() == [64] * 3 and max(spec.lens.tolist()) <= capacity
    assert check_events(dec, spec, events) > 0


def test_a_prompt_without_room_changes_nothing(cuda):
    for kw, P in ((dict(capacity=20), 22), (dict(capacity=60, max_positions=20), 22),
                  (dict(capacity=56, budget=40, recent=12, max_positions=50), 52)):
        dec, spec = make(cuda, parents=[-1, 0], **kw)
        with pytest.raises(ValueError):
            spec.prefill(prompt(cuda, 3, P, 1000), chunk=4)
        assert spec.lens.tolist() == [0] * 3 and spec.history == [[]] * 3
        spec.prefill(prompt(cuda, 3, 9, 1000), chunk=4)
        run_checked(dec, spec, 2, lambda hist, m: [-1] * (m - 1))


def test_a_prompt_after_tokens(cuda):
    """The next turn of a conversation: the last chosen token comes before it."""
    rng = np.random.default_rng(2)
    dec, spec = make(cuda, parents=[-1, 0, 0, 1])
    spec.prefill(prompt(cuda, 3, 7, 1000), chunk=4)
    for P in (1, 6, 9):
        run_checked(dec, spec, 3, lambda hist, m: rng.integers(-1, 1000, m - 1).tolist())
        spec.prefill(prompt(cuda, 3, P, 1000, seed=P), chunk=4)
    run_checked(dec, spec, 3, lambda hist, m: rng.integers(-1, 1000, m - 1).tolist())
    for n, hist in enumerate(spec.history):
        assert int(spec.next_pos[n]) == len(hist) - 1 and int(spec.ids[n]) == hist[-1]


def test_a_prompt_after_a_prompt(cuda):
    dec, spec = make(cuda, parents=[-1, 0])
    ids = prompt(cuda, 3, 12, 1000)
    spec.prefill(ids[:, :1])
    spec.prefill(ids[:, 1:5])
    spec.prefill(ids[:, 5:], chunk=3)
    assert spec.lens.tolist() == [11] * 3 and spec.history == ids.tolist()
    run_checked(dec, spec, 3, lambda hist, m: [-1])


def test_device_errors_are_raised(cuda):
    """A drafted token outside the vocabulary sets the index bit."""
    from moat_b200._lib import MoatError
    dec, spec = make(cuda, parents=[-1, 0])
    spec.prefill(prompt(cuda, 3, 7, 1000))
    spec.generate(2, lambda hist, m: [-1])
    with pytest.raises(MoatError, match="index"):
        spec.generate(2, lambda hist, m: [1000])


def test_device_errors_of_a_prompt_are_raised(cuda):
    from moat_b200._lib import MoatError
    dec, spec = make(cuda, parents=[-1, 0])
    ids = prompt(cuda, 3, 7, 1000)
    ids[1, 3] = 5000
    spec.prefill(ids)
    with pytest.raises(MoatError, match="index"):
        spec.generate(1, lambda hist, m: [-1])
