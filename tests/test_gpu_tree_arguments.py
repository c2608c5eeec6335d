"""Refusals of drafted decoding's entry points: what a kernel would read or write out of place
is an error before anything is launched."""

import pytest

from test_gpu_tree import inputs

pytestmark = pytest.mark.gpu


def accept_args(cuda, T=2, m=4, Hkv=2, Lmax=16, d=64, layers=3):
    import torch
    i = torch.zeros((T, m), dtype=torch.int32, device=cuda)
    n = torch.zeros(T, dtype=torch.int32, device=cuda)
    k = torch.zeros((layers, T, Hkv, Lmax, d), dtype=torch.float16, device=cuda)
    kd = torch.ones((layers, T, m, Hkv, d), dtype=torch.float16, device=cuda)
    return dict(tokens=i, parents=i, target=i, lens=n, next_pos=n, k_cache=k, v_cache=k.clone(), k_draft=kd,
                v_draft=kd.clone())


def test_an_error_word_is_a_32_bit_word(cuda):
    """The kernels set its bits with a 32-bit atomic."""
    import torch
    from moat_b200.tree import accept_tree, tree_attention
    x = inputs(cuda, 2, 4, 8, 2, 64, [5, 9], 16, seed=1)
    a = accept_args(cuda)
    i32 = torch.zeros(4, dtype=torch.int32, device=cuda)
    for err in (i32[:0], i32.view(torch.uint8)[1:2], i32.short(), i32.long(), i32.float(), i32.cpu()):
        with pytest.raises(ValueError, match="dev_err"):
            tree_attention(**x, dev_err=err)
        with pytest.raises(ValueError, match="dev_err"):
            accept_tree(**a, dev_err=err)
    tree_attention(**x, dev_err=i32[1:])
    accept_tree(**a, dev_err=i32[1:])
    assert not bool(i32.any())


def test_what_is_written_is_not_broadcast(cuda):
    """Several CTAs would write one place; what is only read may be broadcast."""
    import torch
    from moat_b200.evict import evict_cache
    from moat_b200.tree import accept_tree, tree_attention
    x = inputs(cuda, 2, 4, 8, 2, 64, [5, 9], 16, seed=1)
    for axis in range(3):
        shape = list(x["q"].shape)
        shape[axis] = 1
        with pytest.raises(ValueError, match="broadcast"):
            tree_attention(**x, out=torch.zeros(shape, dtype=torch.float16, device=cuda).expand(x["q"].shape))
    one = torch.zeros((1, 1, 8, 64), dtype=torch.float16, device=cuda)  # an axis of length 1 may have any stride
    y = inputs(cuda, 1, 1, 8, 2, 64, [5], 16, seed=1)
    tree_attention(**y, out=one.as_strided(one.shape, (0, 0, 64, 1)))
    a = accept_args(cuda)
    s = torch.zeros((3, 2, 2, 16), device=cuda)
    p = torch.zeros((3, 2, 2, 16), dtype=torch.int32, device=cuda)
    for axis in range(4):
        for name in ("k_cache", "v_cache"):
            shape = list(a["k_cache"].shape)
            shape[axis] = 1
            wide = {name: torch.zeros(shape, dtype=torch.float16, device=cuda).expand(a["k_cache"].shape)}
            with pytest.raises(ValueError, match="broadcast"):
                accept_tree(**{**a, **wide})
            caches = {**{n: a[n] for n in ("k_cache", "v_cache")}, **wide}
            with pytest.raises(ValueError, match="broadcast"):
                evict_cache(**caches, scores=s, positions=p, lens=a["lens"], next_pos=a["lens"], budget=8, recent=2)
    draft = a["k_draft"][:1].expand(a["k_draft"].shape)
    accept_tree(**{**a, "k_draft": draft, "tokens": a["tokens"] + 1})
    assert bool((a["k_cache"][:, :, :, 0] == 1).all())


@pytest.mark.parametrize("T,m,H,Hkv,d,lens,Lmax", [(2, 1, 4, 2, 128, [300, 40], 300), (2, 40, 8, 2, 64, [2000, 9], 2000),
                                                   (1, 20, 4, 2, 256, [900], 900), (9, 8, 8, 8, 128, [700] * 9, 700)])
def test_the_output_in_the_queries_place(cuda, T, m, H, Hkv, d, lens, Lmax):
    """Without scores it is the same; with them the weights would read queries that are no longer there."""
    import torch
    from moat_b200.tree import tree_attention
    x = inputs(cuda, T, m, H, Hkv, d, lens, Lmax, seed=2)
    want = tree_attention(**x)
    q = x["q"].clone()
    assert tree_attention(**{**x, "q": q}, out=q) is q and torch.equal(q, want)
    with pytest.raises(ValueError, match="q"):
        tree_attention(**x, out=x["q"], scores=torch.zeros((T, Hkv, Lmax), device=cuda))
