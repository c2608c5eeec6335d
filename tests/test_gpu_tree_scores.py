"""Row weights beside what no node sees: padding nodes' queries, infinite scores. References and
tolerances as in test_gpu_tree.py."""

import pytest

from test_gpu_tree import check, inputs, reference

pytestmark = pytest.mark.gpu

SHAPES = [
    # T, m, H, Hkv, d, lens, Lmax; every third trace has fewer nodes than m, and a node has several heads
    (3, 3, 4, 2, 128, [700, 0, 300], 700),  # kept scores
    (3, 8, 4, 2, 64, [130, 1300, 256], 1300),
    (3, 17, 6, 2, 128, [500, 3, 129], 512),  # formed again
    (3, 63, 16, 2, 64, [33, 0, 900], 901),  # several row blocks
    (3, 5, 4, 2, 200, [40, 600, 300], 600),  # general path
]
ids = dict(ids=lambda s: "x".join(map(str, s[:5])))


@pytest.mark.parametrize("stale", [float("nan"), float("inf"), -float("inf"), 65504.0])
@pytest.mark.parametrize("shape", SHAPES, **ids)
def test_queries_of_padding_nodes_do_not_matter(cuda, shape, stale):
    x = inputs(cuda, *shape, seed=3, padded=True, stale=stale)
    padding = x["masks"] == 0
    assert bool(padding.any())
    x["q"][padding] = stale
    check(x, weights=True)


@pytest.mark.parametrize("shape", SHAPES, **ids)
def test_a_key_that_weighs_nothing(cuda, shape):
    """A cached key with an infinite element whose score is -inf for every node: its weight is 0."""
    import torch
    from moat_b200.tree import tree_attention
    x = inputs(cuda, *shape, seed=4, padded=True)
    T, m, H, Hkv, d, lens, Lmax = shape
    rel = reference(x)[4]
    x["q"][..., 5] = x["q"][..., 5].abs() + 0.5
    for t, n in enumerate(lens):
        if n > 0:
            x["k_cache"][t, :, n // 2, 5] = -float("inf")
    ref, tol, wc, wd, _ = reference(x)
    out, so, ds = tree_attention(**x, scores=torch.zeros((T, Hkv, Lmax), device=cuda))
    assert bool(((out.double() - ref).abs() <= tol).all())
    assert bool(((so.double() - wc).abs() <= 2 * rel * wc + 1e-30).all())  # the queries grew by less than that
    assert bool(((ds.double() - wd).abs() <= 2 * rel * wd + 1e-30).all())
    for t, n in enumerate(lens):
        assert n == 0 or bool((so[t, :, n // 2] == 0).all())


@pytest.mark.parametrize("m,H,Hkv,d,n", [(3, 4, 2, 128, 300), (7, 4, 2, 64, 40), (9, 16, 2, 128, 700), (5, 4, 2, 200, 90)])
def test_an_infinite_score_reaches_only_the_rows_that_its_node_sees(cuda, m, H, Hkv, d, n):
    """Node 1's own key gives it a score of +inf, so what it weighs is not a number; node 2, its
    sibling, is not seen by it: that row's weight is its own nodes'."""
    import torch
    from moat_b200.tree import tree_attention, tree_masks
    x = inputs(cuda, 2, m, H, Hkv, d, [n, 0], n, seed=m)
    x["masks"] = torch.from_numpy(tree_masks([-1, 0, 0] + [2] * (m - 3))).to(cuda)
    rel = reference(x)[4]
    x["q"][..., 5] = x["q"][..., 5].abs() + 0.5
    clean = {**x, "masks": x["masks"].clone()}
    clean["masks"][1] = 0
    wd = reference(clean)[3]
    x["k_draft"][:, 1, :, 5] = float("inf")
    out, so, ds = tree_attention(**x, scores=torch.zeros((2, Hkv, n), device=cuda))
    assert not bool(torch.isfinite(out[:, 1]).any()) and bool(torch.isfinite(out[:, 2:]).all())
    assert bool(torch.isnan(so[0]).all()) and bool(torch.isnan(ds[..., :2]).all())
    assert bool(((ds.double() - wd).abs() <= 2 * rel * wd + 1e-30)[..., 2:].all())


@pytest.mark.parametrize("T,m,H,Hkv,d", [(1, 1, 1, 1, 64), (2, 5, 4, 2, 128), (2, 33, 8, 2, 64), (1, 3, 2, 1, 33)])
def test_weights_without_a_cache(cuda, T, m, H, Hkv, d):
    """Lmax = 0: there is nothing but the draft."""
    check(inputs(cuda, T, m, H, Hkv, d, [0] * T, 0, seed=m), weights=True)
