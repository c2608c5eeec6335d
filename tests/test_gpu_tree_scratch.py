"""Scratch of drafted decoding's calls: it returns to torch's allocator, and graphs share none."""

import pytest

from test_gpu_tree import inputs

pytestmark = pytest.mark.gpu


def evict_args(cuda, T=2, Hkv=4, n=9000, d=64):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(T)
    k, v = (torch.randn((T, Hkv, n, d), generator=g, device=cuda).half() for _ in range(2))
    return dict(k_cache=k, v_cache=v, scores=torch.rand((T, Hkv, n), generator=g, device=cuda),
                positions=torch.arange(n, dtype=torch.int32, device=cuda).repeat(T, Hkv, 1),
                lens=torch.tensor([n - t for t in range(T)], dtype=torch.int32, device=cuda),
                next_pos=torch.full((T,), n, dtype=torch.int32, device=cuda))


def test_scratch_is_given_back(cuda):
    """Kept scores of 16 rows are some 40 MB here; after the call none of them is held."""
    import torch
    from moat_b200.evict import evict_cache
    from moat_b200.tree import tree_attention
    x = inputs(cuda, 4, 2, 64, 8, 64, [20000, 3, 15001, 77], 20000, seed=1)
    s = torch.zeros((4, 8, 20000), device=cuda)
    e = evict_args(cuda)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    tree_attention(**x, scores=s)
    assert torch.cuda.max_memory_allocated() - before > 40 << 20
    evict_cache(**e, budget=4000, recent=100)
    assert torch.cuda.memory_allocated() == before


def test_graphs_captured_on_one_stream_replay_side_by_side(cuda):
    """Two captures (torch's capture stream is the same for both), replayed on two streams at once."""
    import torch
    from moat_b200.evict import evict_cache
    from moat_b200.tree import tree_attention
    cases = [inputs(cuda, 2, 16, 16, 4, 128, [5000 - 7 * i, 333], 5000, seed=20 + i) for i in range(2)]
    scores = [torch.rand((2, 4, 5000), device=cuda) for _ in range(2)]
    evictions = [evict_args(cuda, T) for T in (2, 3)]
    eager = []
    for x, s, e in zip(cases, scores, evictions):
        e = {**e, "k_cache": e["k_cache"].clone(), "v_cache": e["v_cache"].clone()}
        out = tree_attention(**x, scores=s, scores_out=torch.zeros_like(s))
        so, po, _ = evict_cache(**e, budget=4000, recent=100, scores_out=torch.zeros_like(e["scores"]),
                                positions_out=torch.zeros_like(e["positions"]))
        eager.append((*out, so, po, e["k_cache"], e["v_cache"]))
    graphs, got = [], []
    for x, s, e in zip(cases, scores, evictions):
        so, eo, po = torch.zeros_like(s), torch.zeros_like(e["scores"]), torch.zeros_like(e["positions"])
        out, ds = torch.zeros_like(x["q"]), torch.zeros((2, 4, 16), device=cuda)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(4):
                tree_attention(**x, out=out, scores=s, scores_out=so, draft_scores=ds)
            evict_cache(**e, budget=4000, recent=100, scores_out=eo, positions_out=po)
        graphs.append(g)
        got.append((out, so, ds, eo, po, e["k_cache"], e["v_cache"]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(25):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_scratch_beyond_the_memory_is_torchs_error(cuda):
    """400 MB of kept scores where the process may have 100 MB more than it has."""
    import torch
    from moat_b200.tree import tree_attention
    torch.cuda.empty_cache()
    x = inputs(cuda, 4, 2, 64, 8, 64, [3] * 4, 8, seed=1)
    for name in ("k_cache", "v_cache"):  # without temporaries, whose place could hold the scratch
        x[name] = torch.zeros((4, 8, 200000, 64), dtype=torch.float16, device=cuda)
    s = torch.zeros((4, 8, 200000), device=cuda)
    torch.cuda.synchronize()
    total = torch.cuda.get_device_properties(cuda).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (100 << 20)) / total, cuda)
        with pytest.raises(torch.OutOfMemoryError):
            tree_attention(**x, scores=s)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, cuda)
    assert tree_attention(**x, scores=s)[1] is s
