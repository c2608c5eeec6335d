"""Attention, weights and eviction one after the other on a stream: every call sees what the one
before it wrote, however the attention shares out its units.

The lengths are those for which the units stay whole, so that the join between the attention and
the weights has nothing to do. Tolerances as in test_gpu_tree.py.
"""

import numpy as np
import pytest

from test_gpu_evict import keep_rows
from test_gpu_tree import inputs, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,m,H,Hkv,lens,Lmax", [
    (40, 1, 8, 8, [600 - 13 * t for t in range(40)], 640),  # more units than SMs
    (40, 3, 24, 8, [600 - 13 * t for t in range(40)], 640),
    (12, 24, 8, 8, [700 - 31 * t for t in range(12)], 1024),  # fewer, scores formed again
    (130, 2, 2, 2, [560 - 4 * t for t in range(130)], 576),  # two launches
    (130, 20, 2, 2, [560 - 4 * t for t in range(130)], 576),  # and scores formed again
    (130, 2, 2, 2, [6000 if t in (3, 128) else 17 for t in range(130)], 6000),  # units cut in either
    (130, 9, 4, 2, [6000 if t in (3, 128) else 17 for t in range(130)], 6000),
])
def test_eviction_right_after_attention(cuda, T, m, H, Hkv, lens, Lmax):
    import torch
    from moat_b200.evict import evict_cache
    from moat_b200.tree import tree_attention
    budget, recent, sinks = 64, 16, 2
    x = inputs(cuda, T, m, H, Hkv, 128, lens, Lmax, seed=T)
    ref, tol, wc, wd, rel = reference(x)
    scores = torch.rand((T, Hkv, Lmax), device=cuda)
    pos = torch.arange(Lmax, dtype=torch.int32, device=cuda).repeat(T, Hkv, 1)
    kept = torch.tensor([min(n, budget) for n in lens], device=cuda).view(T, 1, 1)
    first = None
    for _ in range(6):
        k, v = x["k_cache"].clone(), x["v_cache"].clone()
        so, so2, po = torch.zeros_like(scores), torch.zeros_like(scores), torch.zeros_like(pos)
        out, _, ds = tree_attention(**{**x, "k_cache": k, "v_cache": v}, scores=scores, scores_out=so)
        _, _, new = evict_cache(k, v, so, pos, x["lens"], x["lens"], budget, recent=recent, sinks=sinks,
                                scores_out=so2, positions_out=po)
        got = (out, so, ds, so2, po, new, k, v)
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    out, so, ds, so2, po, new, k, v = first
    assert bool(((out.double() - ref).abs() <= tol).all())
    valid = torch.arange(Lmax, device=cuda) < x["lens"].view(T, 1, 1)
    want = torch.where(valid, scores.double() + wc, 0.0)
    assert bool(((so.double() - want).abs() <= rel * wc + 2.0 ** -23 * want.abs()).all())
    assert bool(((ds.double() - wd).abs() <= rel * wd + 1e-30).all())
    assert new.tolist() == kept.flatten().tolist()
    so, pos, so2, po = (t.cpu().numpy() for t in (so, pos, so2, po))
    for t, n in enumerate(lens):
        for h in range(Hkv):
            src = keep_rows(so[t, h], pos[t, h], n, n, budget, recent, sinks)
            np.testing.assert_array_equal(so2[t, h, :len(src)], so[t, h, src])
            np.testing.assert_array_equal(po[t, h, :len(src)], src)
            assert torch.equal(k[t, h, :len(src)], x["k_cache"][t, h, torch.from_numpy(src).to(cuda)])
            assert torch.equal(v[t, h, :len(src)], x["v_cache"][t, h, torch.from_numpy(src).to(cuda)])
