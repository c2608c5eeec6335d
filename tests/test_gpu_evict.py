"""GPU eviction against a plain host implementation: everything is selection and copies,
so every value has to be equal."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def keep_rows(score, pos, n, next_pos, budget, recent, sinks):
    """Source row of every kept row of one (layer, trace, head), on the host."""
    kept = min(n, budget)
    p, s = pos[:n].astype(np.int64), score[:n].astype(np.float64)
    safe = (p >= next_pos - recent) | (p < sinks)
    s = np.where(safe, 0.0, np.where(np.isnan(s), -np.inf, s)) + 0.0  # guarded rows rank alike, whatever they scored
    order = np.lexsort((np.arange(n), -s, ~safe & np.isnan(score[:n]), ~safe))  # guarded, NaN last, score, row
    inside = np.zeros(n, bool)
    inside[order[:kept]] = True
    src = np.arange(kept)
    src[~inside[:kept]] = kept + np.flatnonzero(inside[kept:])
    return src


def run(cuda, layers, T, Hkv, Lmax, d, lens, budget, recent, sinks, scores=None, positions=None, in_place=False,
        seed=0, cache=None):
    import torch
    from moat_b200.evict import evict_cache
    rng = np.random.default_rng(seed)
    lead = () if layers is None else (layers,)
    full = lead + (T, Hkv, Lmax)
    if scores is None:
        scores = np.where(rng.random(full) < 0.3, 0.0, rng.lognormal(0, 2, full)).astype(np.float32)
    if positions is None:
        positions = np.argsort(rng.random(full), axis=-1).astype(np.int32)
    next_pos = np.asarray([n for n in lens], np.int32)
    if cache is None:
        k, v = (torch.randn(full + (d,), device=cuda).half() for _ in range(2))
    else:
        k, v = cache
    k0, v0 = k.cpu(), v.cpu()
    s, p = torch.from_numpy(scores.copy()).to(cuda), torch.from_numpy(positions.copy()).to(cuda)
    so, po = (s, p) if in_place else (torch.full_like(s, -3.0), torch.full_like(p, -3))
    ln, nx = torch.tensor(lens, dtype=torch.int32, device=cuda), torch.from_numpy(next_pos).to(cuda)
    s2, p2, new = evict_cache(k, v, s, p, ln, nx, budget, recent=recent, sinks=sinks,
                              scores_out=None if in_place else so, positions_out=None if in_place else po)
    assert s2 is so and p2 is po
    assert new.tolist() == [min(max(n, 0), Lmax, budget) for n in lens] and ln.tolist() == list(lens)
    k, v, so, po = k.cpu(), v.cpu(), so.cpu().numpy(), po.cpu().numpy()
    for at in np.ndindex(*full[:-1]):
        t = at[-2]
        n = min(max(lens[t], 0), Lmax)
        src = keep_rows(scores[at], positions[at], n, int(next_pos[t]), budget, recent, sinks)
        c = len(src)
        np.testing.assert_array_equal(so[at][:c], scores[at][src])
        np.testing.assert_array_equal(po[at][:c], positions[at][src])
        np.testing.assert_array_equal(so[at][c:], scores[at][c:] if in_place else -3.0)
        for new_rows, old in ((k[at], k0[at]), (v[at], v0[at])):
            assert torch.equal(new_rows[:c].view(torch.int16), old[src].view(torch.int16))
            assert torch.equal(new_rows[c:].view(torch.int16), old[c:].view(torch.int16))  # rows beyond: untouched
    return so, po


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layers,T,Hkv,Lmax,d,lens,budget,recent,sinks", [
    (None, 1, 1, 1, 64, [1], 1, 0, 0),
    (None, 1, 2, 5, 64, [5], 1, 1, 0),
    (None, 3, 2, 40, 64, [0, 17, 40], 16, 4, 2),
    (2, 2, 3, 300, 128, [300, 257], 256, 32, 4),
    (1, 2, 1, 1100, 72, [1025, 1024], 100, 50, 50),
    (1, 1, 2, 2049, 64, [2049], 2048, 2000, 0),
    (1, 1, 1, 5000, 33, [4999], 3333, 10, 1),
    (3, 2, 2, 130, 80, [130, 129], 129, 0, 0),
    (1, 1, 2, 70000, 64, [69999], 20000, 300, 4),
    (40, 1, 8, 1500, 64, [1400], 700, 64, 4),  # the units alone fill the GPU
    (1, 2, 40, 9000, 64, [8999, 7000], 4000, 100, 4),
    (1, 1, 1, 400003, 8, [400001], 150000, 300, 4),
])
def test_evict(cuda, layers, T, Hkv, Lmax, d, lens, budget, recent, sinks, in_place):
    run(cuda, layers, T, Hkv, Lmax, d, lens, budget, recent, sinks, in_place=in_place, seed=Lmax)


def test_ties_signed_zeros_infinities_and_nan(cuda):
    rng = np.random.default_rng(1)
    full = (2, 2, 600)
    values = np.array([0.0, -0.0, 1.0, -1.0, np.inf, -np.inf, np.nan, 1e-45, -1e-45, 3.4e38], np.float32)
    for seed in range(4):
        scores = values[rng.integers(0, len(values), full)]
        run(cuda, None, 2, 2, 600, 64, [600, 480], 300, 20, 2, scores=scores, seed=seed)


def test_all_scores_equal_keeps_the_lowest_rows(cuda):
    scores = np.zeros((1, 1, 4000), np.float32)
    so, po = run(cuda, None, 1, 1, 4000, 64, [4000], 1500, 0, 0, scores=scores)
    pos = np.argsort(np.random.default_rng(0).random((1, 1, 4000)), axis=-1)  # not sorted: rows decide, not positions
    assert po.shape == pos.shape


def test_more_guarded_rows_than_budget(cuda):
    """Positions that repeat can guard more rows than the budget: the lowest rows stay."""
    pos = np.full((1, 1, 500), 499, np.int32)
    run(cuda, None, 1, 1, 500, 64, [500], 100, 50, 0, positions=pos)


def test_lengths_out_of_range_are_clamped(cuda):
    run(cuda, None, 3, 1, 64, 64, [-3, 90, 64], 20, 5, 1)


def test_strided_caches(cuda):
    import torch
    k = torch.randn((2, 2, 210, 3, 64), device=cuda).half().transpose(2, 3)
    v = torch.randn((2, 2, 3, 210, 65), device=cuda).half()[..., :64]
    run(cuda, 2, 2, 3, 210, 64, [210, 150], 100, 10, 2, cache=(k, v))


def test_repeated_call_changes_nothing_more(cuda):
    """Out of place, the caches' moves are idempotent: no row is both read and written."""
    import torch
    from moat_b200.evict import evict_cache
    k, v = (torch.randn((2, 4, 500, 64), device=cuda).half() for _ in range(2))
    s = torch.rand((2, 4, 500), device=cuda)
    p = torch.arange(500, dtype=torch.int32, device=cuda).repeat(2, 4, 1)
    n = torch.tensor([500, 333], dtype=torch.int32, device=cuda)
    outs = []
    for _ in range(3):
        so, po, ln = evict_cache(k, v, s, p, n, n, 200, recent=20, sinks=4, scores_out=torch.zeros_like(s),
                                 positions_out=torch.zeros_like(p))
        outs.append((so, po, ln, k.clone(), v.clone()))
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], o))


def test_attention_is_the_same_in_any_row_order(cuda):
    """Evicting rows that carry no weight leaves the attention as it was (to the rounding
    of another order of summation: 2 units in the last place of fp16, of values below 4)."""
    import torch
    from moat_b200.evict import evict_cache
    from moat_b200.tree import tree_attention
    g = torch.Generator(device=cuda)
    g.manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda).half()  # noqa: E731
    q, kd, vd, k, v = rnd(1, 2, 4, 64), rnd(1, 2, 2, 64), rnd(1, 2, 2, 64), rnd(1, 2, 300, 64), rnd(1, 2, 300, 64)
    q[..., 0] = 30.0
    dead = torch.randperm(280, generator=g, device=cuda)[:100]
    k[:, :, :, 0] = 0.0
    k[:, :, dead, 0] = -60.0  # scores near -225: a weight of exactly 0 in fp32
    masks = torch.tensor([1, 3], dtype=torch.int64, device=cuda)
    n = torch.tensor([300], dtype=torch.int32, device=cuda)
    pos = torch.arange(300, dtype=torch.int32, device=cuda).repeat(1, 2, 1)
    before, s, _ = tree_attention(q, k, v, n, kd, vd, masks, scores=torch.zeros((1, 2, 300), device=cuda))
    assert bool((s[:, :, dead] == 0).all())
    s, pos, n = evict_cache(k, v, s, pos, n, n, 200, recent=20, sinks=0)
    assert n.tolist() == [200] and bool((s[..., :200] > 0).all())
    assert set(pos[0, 0, :200].tolist()) == set(range(300)) - set(dead.tolist())
    after = tree_attention(q, k, v, n, kd, vd, masks)
    assert float((after.float() - before.float()).abs().max()) <= 4 * 2.0 ** -10


def test_refusals(cuda):
    import torch
    from moat_b200.evict import evict_cache
    k = torch.zeros((1, 2, 32, 64), dtype=torch.float16, device=cuda)
    s = torch.zeros((1, 2, 32), device=cuda)
    p = torch.zeros((1, 2, 32), dtype=torch.int32, device=cuda)
    n = torch.tensor([32], dtype=torch.int32, device=cuda)
    base = dict(k_cache=k, v_cache=k.clone(), scores=s, positions=p, lens=n, next_pos=n, budget=16, recent=4, sinks=2)
    for change in (dict(budget=0), dict(budget=5), dict(recent=-1), dict(sinks=-1), dict(lens=n.long()),
                   dict(scores=s.half()), dict(positions=p.long()), dict(scores=s[:, :, :31]), dict(v_cache=k.float()),
                   dict(v_cache=k[:, :, :31]), dict(k_cache=k[0]), dict(k_cache=k.cpu()),
                   dict(scores_out=torch.zeros_like(s)), dict(k_cache=k.transpose(2, 3))):
        with pytest.raises(ValueError):
            evict_cache(**{**base, **change})
    with pytest.raises(TypeError):
        evict_cache(**{**base, "k_cache": k.cpu().numpy()})
