"""GPU parity of drafted decoding's attention and acceptance with plain 64-bit
implementations.

Tolerances, with u the unit roundoff of the element type (2^-11 fp16, 2^-8 bf16):
an output is sum_l p_l v_l / sum_l p_l with every p_l rounded once (relative u, or 2^-25 of
the row's largest weight in fp16's subnormals) and the result rounded once, so
|error| <= 1.1 u (sum p |v| + |out|) + 2^-24 L max|v|, plus fp32 work far below that.
A row's weight is a sum of fp32 exponentials of scores whose error is at most
2 d 2^-24 S, S = scale log2(e) sum_c |q_c k_c| (any order of fp32 sums, truncated or not);
it enters once through the score and once through the row's normaliser.
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def random_parents(rng, T, m, nodes=None):
    out = np.full((T, m), -1)
    for t in range(T):
        for i in range(1, m if nodes is None else nodes[t]):
            out[t, i] = rng.integers(max(0, i - 5), i)
    return out


def inputs(cuda, T, m, H, Hkv, d, lens, Lmax, dtype="float16", seed=0, padded=False, stale=None):
    import torch
    from moat_b200.tree import tree_masks
    dt = getattr(torch, dtype)
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=cuda).to(dt)

    rng = np.random.default_rng(seed)
    nodes = [max(1, m - t % 3) for t in range(T)] if padded else None
    masks = tree_masks(random_parents(rng, T, m, nodes))
    x = {"q": normal(T, m, H, d), "k_cache": normal(T, Hkv, Lmax, d), "v_cache": normal(T, Hkv, Lmax, d),
         "lens": torch.tensor(lens, dtype=torch.int32, device=cuda), "k_draft": normal(T, m, Hkv, d),
         "v_draft": normal(T, m, Hkv, d), "masks": torch.from_numpy(masks).to(cuda)}
    if stale is not None:  # what rows beyond the valid ones, and padding nodes, may hold
        for t in range(T):
            x["k_cache"][t, :, max(0, lens[t]):] = stale
            x["v_cache"][t, :, max(0, lens[t]):] = stale
            for i in range(m):
                if masks[t, i] == 0:
                    x["k_draft"][t, i] = stale
                    x["v_draft"][t, i] = stale
    return x


def reference(x, scale=None):
    """out, its tolerance, the weights of the cached rows and of the draft's, and their
    relative tolerance, in float64 on the GPU."""
    import torch
    q, T, m, H, d = x["q"], *x["q"].shape
    Hkv, Lmax = x["k_cache"].shape[1:3]
    G = H // Hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u = U[str(q.dtype).split(".")[1]]
    masks = x["masks"].cpu().numpy().view(np.uint64)
    masks = np.broadcast_to(masks, (T, m))
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    wc = torch.zeros((T, Hkv, Lmax), dtype=torch.float64, device=q.device)
    wd = torch.zeros((T, Hkv, m), dtype=torch.float64, device=q.device)
    rel = 0.0
    for t in range(T):
        n = min(max(int(x["lens"][t]), 0), Lmax)
        for i in range(m):
            nodes = [j for j in range(m) if (int(masks[t, i]) >> j) & 1]
            if not nodes:
                continue
            for h in range(H):
                kv = h // G
                k = torch.cat([x["k_cache"][t, kv, :n], x["k_draft"][t, nodes, kv]]).double()
                v = torch.cat([x["v_cache"][t, kv, :n], x["v_draft"][t, nodes, kv]]).double()
                qr = q[t, i, h].double()
                p = torch.softmax(scale * (k @ qr), 0)
                out[t, i, h] = p @ v
                tol[t, i, h] = (1.1 * u * (p @ v.abs() + out[t, i, h].abs()) + 2.0 ** -24 * len(p) * v.abs().max()
                                + 1e-6)
                wc[t, kv, :n] += p[:n]
                wd[t, kv, nodes] += p[n:]
                size = abs(scale) * 1.4427 * float((k.abs() @ qr.abs()).max())
                rel = max(rel, 2 * 0.6931 * 2 * d * 2.0 ** -24 * size + 2.0 ** -20)
    return out, tol, wc, wd, rel


def check(x, weights=False, scale=None, **kw):
    import torch
    from moat_b200.tree import tree_attention
    ref, tol, wc, wd, rel = reference(x, scale)
    dev_err = torch.zeros(1, dtype=torch.int32, device=ref.device)
    kw["dev_err"] = dev_err
    if not weights:
        got = tree_attention(**x, scale=scale, **kw)
    else:
        T, Hkv, Lmax = x["k_cache"].shape[:3]
        scores = torch.rand((T, Hkv, Lmax), device=ref.device)
        old = scores.clone()
        got, so, ds = tree_attention(**x, scale=scale, scores=scores, **kw)
        assert so is scores
        n = x["lens"].clamp(0, Lmax).view(T, 1, 1)
        valid = torch.arange(Lmax, device=ref.device) < n
        assert torch.equal(so[~valid.expand_as(so)], old[~valid.expand_as(so)])  # rows beyond the valid ones: untouched
        want = torch.where(valid, old.double() + wc, old.double())
        assert bool(((so.double() - want).abs() <= rel * wc + 2.0 ** -23 * want.abs()).all())
        assert bool(((ds.double() - wd).abs() <= rel * wd + 1e-30).all())
    assert int(dev_err) == 0  # no bounded wait gave up
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"largest error over tolerance {(err / tol.clamp(min=1e-30)).max().item():.3g}"
    assert bool((got[tol.sum(-1) == 0] == 0).all())  # padding
    return got


SHAPES = [
    # T, m, H, Hkv, d, lens, Lmax
    (1, 1, 1, 1, 64, [0], 0),
    (1, 1, 1, 1, 128, [1], 1),
    (2, 1, 4, 4, 128, [127, 128], 130),
    (3, 2, 4, 2, 64, [0, 129, 300], 300),
    (2, 8, 8, 2, 128, [255, 256], 257),
    (2, 17, 6, 2, 128, [500, 3], 512),
    (1, 64, 4, 2, 64, [1000], 1024),
    (2, 63, 16, 2, 64, [33, 0], 64),
    (1, 5, 8, 1, 96, [700], 701),
    (1, 33, 12, 4, 80, [161], 200),
    (2, 3, 5, 5, 8, [40, 77], 77),
    (1, 4, 4, 2, 40, [600], 600),
    (1, 9, 4, 4, 256, [400], 400),
    (1, 3, 2, 1, 33, [90], 100),
    (1, 1, 8, 1, 128, [5000], 5001),
    (5, 16, 32, 8, 128, [1, 1025, 64, 0, 2000], 2048),
    (16, 1, 16, 16, 128, [1100 - 67 * t for t in range(16)], 1100),  # several odd-length pieces per CTA
    (6, 40, 16, 2, 64, [130, 1300, 700, 0, 901, 2500], 2500),  # row blocks and such pieces
    (80, 1, 8, 8, 128, [400 - 3 * t for t in range(79)] + [0], 400),  # more units than SMs: dealt out whole
    (16, 2, 8, 8, 128, [2000 - t for t in range(16)], 2000),  # as many units as SMs, nearly: one each
    (16, 5, 32, 8, 128, [4100 - t for t in range(16)], 4100),  # the same with more than 16 rows
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])))
def test_attention(cuda, shape, dtype):
    check(inputs(cuda, *shape, dtype=dtype, seed=sum(shape[:5])))


@pytest.mark.parametrize("shape", SHAPES[1:], ids=lambda s: "x".join(map(str, s[:5])))
def test_attention_with_scores(cuda, shape):
    check(inputs(cuda, *shape, seed=sum(shape[:5]) + 1, padded=True), weights=True)


@pytest.mark.parametrize("stale", [float("nan"), float("inf"), -65504.0])
@pytest.mark.parametrize("shape", [SHAPES[3], SHAPES[5], SHAPES[7], SHAPES[11]], ids=lambda s: "x".join(map(str, s[:5])))
def test_rows_that_no_node_sees_do_not_matter(cuda, shape, stale):
    check(inputs(cuda, *shape, seed=3, padded=True, stale=stale), weights=True)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("T,m,H,Hkv,d,lens,Lmax", [(2, 7, 4, 2, 128, [40, 300], 300), (2, 40, 8, 2, 64, [0, 1500], 1500),
                                                   (2, 5, 4, 2, 33, [40, 200], 200), (2, 9, 2, 2, 96, [9, 2600], 2600)])
def test_values_that_are_not_finite_reach_only_who_sees_them(cuda, T, m, H, Hkv, d, lens, Lmax, bad, dtype):
    """One value of one drafted row (and, in another run, one of its key's): the nodes that
    see the row get NaN or the infinity there, every other output is what it was."""
    import torch
    from moat_b200.tree import tree_attention
    x = inputs(cuda, T, m, H, Hkv, d, lens, Lmax, dtype=dtype, seed=m)
    node, c = m // 3, d - 3
    sees = ((x["masks"] >> node) & 1).bool()  # [T, m]
    assert bool(sees.any()) and not bool(sees.all())
    clean = tree_attention(**x)
    v = x["v_draft"].clone()
    v[:, node, :, c] = bad
    got = tree_attention(**{**x, "v_draft": v})
    assert not bool(torch.isfinite(got[sees][..., c]).any())
    if not math.isnan(bad):
        assert bool((got[sees][..., c] == bad).all())
    rest = torch.ones(got.shape, dtype=torch.bool, device=cuda)
    rest[..., c] = ~sees.unsqueeze(-1)
    assert torch.equal(got[rest], clean[rest])
    k = x["k_draft"].clone()
    k[:, node, :, c] = float("nan")
    scores = torch.zeros((T, Hkv, Lmax), device=cuda)
    got, so, ds = tree_attention(**{**x, "k_draft": k}, scores=scores)
    assert bool(torch.isnan(got[sees]).all())
    ref, tol = reference(x)[:2]  # a row's rounding may depend on the others' maxima
    assert bool(((got.double() - ref).abs()[~sees] <= tol[~sees]).all())


@pytest.mark.parametrize("m,H,Hkv", [(7, 8, 8), (12, 16, 8)])
def test_values_that_are_not_finite_stay_in_their_trace(cuda, m, H, Hkv):
    """Many traces without cached rows (one tile each, several per CTA); every other one has a
    NaN in one drafted row, another row in each."""
    import torch
    from moat_b200.tree import tree_attention
    T, d = 101, 128
    x = inputs(cuda, T, m, H, Hkv, d, [0] * T, 8, seed=m)
    clean = tree_attention(**x)
    v, rest = x["v_draft"].clone(), torch.ones(clean.shape, dtype=torch.bool, device=cuda)
    for t in range(0, T, 2):
        v[t, t % m, :, t % d] = float("nan")
        rest[t, :, :, t % d] = ~((x["masks"][t] >> (t % m)) & 1).bool().unsqueeze(-1)
    for _ in range(20):
        got = tree_attention(**{**x, "v_draft": v})
        assert bool(torch.isnan(got[~rest]).all())
        assert torch.equal(got[rest], clean[rest])


def test_lengths_out_of_range_are_clamped(cuda):
    x = inputs(cuda, 3, 2, 4, 2, 64, [-5, 70, 64], 64, seed=4)
    check(x, weights=True)


def test_large_scores_and_late_maxima(cuda):
    """Scores of several hundred, the largest at the very end, at the start, and in the draft."""
    for where in ("end", "start", "draft"):
        x = inputs(cuda, 2, 4, 8, 2, 128, [900, 640], 900, seed=5)
        big = x["q"][:, 0, ::4] * 3.0  # [T, Hkv, d]
        if where == "draft":
            x["k_draft"][:, 2] = big
        else:
            for t, n in enumerate([900, 640]):
                x["k_cache"][t, :, n - 1 if where == "end" else 0] = big[t]
        x["q"] *= 4
        check(x, weights=True)


def test_very_negative_scores(cuda):
    """All scores far below zero: the softmax is still normalised by its own maximum."""
    x = inputs(cuda, 1, 3, 4, 2, 64, [300], 300, seed=6)
    x["q"][:] = 8.0
    x["k_cache"][:] = -8.0 + 0.1 * x["k_cache"]
    x["k_draft"][:] = -8.0
    check(x, weights=True)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.125])
def test_scale(cuda, scale):
    check(inputs(cuda, 2, 5, 8, 2, 64, [200, 17], 256, seed=7), weights=True, scale=scale)


@pytest.mark.parametrize("d", [64, 128])
def test_strides_and_alignment(cuda, d):
    """Caches laid out [T, L, Hkv, d], drafts as slices of one projection, rows padded by 8
    and by 1 elements, a base address off 16 bytes, a strided output."""
    import torch
    T, m, H, Hkv, Lmax, lens = 2, 7, 8, 2, 333, [333, 130]
    base = inputs(cuda, T, m, H, Hkv, d, lens, Lmax, seed=8)

    def check_variant(**change):
        return check({**base, **change}, weights=True)

    first = check_variant()
    permuted = {n: base[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("k_cache", "v_cache")}
    assert torch.equal(first, check_variant(**permuted))
    qkv = torch.cat([base[n].reshape(T, m, -1) for n in ("q", "k_draft", "v_draft")], 2)
    cut = qkv.split([H * d, Hkv * d, Hkv * d], 2)
    assert torch.equal(first, check_variant(q=cut[0].view(T, m, H, d), k_draft=cut[1].view(T, m, Hkv, d),
                                            v_draft=cut[2].view(T, m, Hkv, d)))
    for pad in (8, 1):
        wide = torch.full((T, Hkv, Lmax, d + pad), float("nan"), dtype=torch.float16, device=cuda)
        wide[..., :d] = base["k_cache"]
        check_variant(k_cache=wide[..., :d])
    for name in ("q", "k_cache", "v_draft"):
        flat = torch.empty(base[name].numel() + 1, dtype=torch.float16, device=cuda)
        odd = flat[1:].view(base[name].shape)
        odd.copy_(base[name])
        check_variant(**{name: odd})
    out = torch.full((T, m, H, 2 * d), 7.0, dtype=torch.float16, device=cuda)
    got = check(base, out=out[..., :d])
    assert got.data_ptr() == out.data_ptr() and bool((out[..., d:] == 7.0).all())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("T,m,H,Hkv,d,lens,Lmax", [(1, 1, 2, 2, 256, [5000], 5000), (3, 5, 6, 2, 200, [3000, 0, 257], 3001),
                                                   (2, 3, 2, 1, 1, [600, 511], 600), (2, 2, 150, 1, 64, [300, 128], 300),
                                                   (1, 64, 4, 1, 77, [1025], 1100)])
def test_general_path_with_spans_of_the_keys(cuda, T, m, H, Hkv, d, lens, Lmax, dtype):
    """Head dims and groups that the tensor cores do not take; long caches cut into spans, some
    of which a short trace leaves empty."""
    import torch
    x = inputs(cuda, T, m, H, Hkv, d, lens, Lmax, dtype=dtype, seed=m + d)
    x["masks"][-1, m // 2] = 0  # a node that sees nothing
    first = check(x, weights=True)
    assert torch.equal(first, check(x))
    assert bool((first[-1, m // 2] == 0).all())


def test_one_tree_for_all_traces(cuda):
    import torch
    x = inputs(cuda, 3, 6, 4, 4, 64, [5, 200, 131], 200, seed=9)
    x["masks"] = x["masks"][1].contiguous()
    one = check(x, weights=True)
    x["masks"] = x["masks"].repeat(3, 1).contiguous()
    assert torch.equal(one, check(x, weights=True))


def test_single_token_of_an_empty_cache_is_its_own_value(cuda):
    import torch
    from moat_b200.tree import tree_attention
    x = inputs(cuda, 2, 1, 4, 2, 128, [0, 0], 16, seed=10)
    got = tree_attention(**x)
    assert torch.equal(got, x["v_draft"].repeat_interleave(2, dim=2))


def test_repeats_bit_for_bit_and_out_of_place_scores(cuda):
    import torch
    from moat_b200.tree import tree_attention
    x = inputs(cuda, 4, 12, 16, 4, 128, [3000, 17, 1500, 900], 3000, seed=11)
    s = torch.rand((4, 4, 3000), device=cuda)
    keep = s.clone()
    runs = []
    for _ in range(3):
        so, ds = torch.zeros_like(s), torch.empty((4, 4, 12), device=cuda)
        out, a, b = tree_attention(**x, scores=s, scores_out=so, draft_scores=ds)
        assert a is so and b is ds
        runs.append((out, so, ds))
    assert torch.equal(s, keep)
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
    # total weight: one per real (node, head)
    total = (runs[0][1] - torch.where(runs[0][1] != 0, s, 0.0)).double().sum() + runs[0][2].double().sum()
    assert abs(total.item() - 4 * 12 * 16) < 1e-2


def test_another_stream_and_graph_replay(cuda):
    import torch
    from moat_b200.tree import tree_attention
    x = inputs(cuda, 2, 8, 8, 2, 128, [700, 90], 1024, seed=12)
    want = tree_attention(**x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = tree_attention(**x)
        g = torch.cuda.CUDAGraph()
        out = torch.empty_like(want)
        with torch.cuda.graph(g, stream=side):
            tree_attention(**x, out=out)
    side.synchronize()
    assert torch.equal(got, want)
    x["lens"].copy_(torch.tensor([100, 1024], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, tree_attention(**x))  # the lengths are read on the device


def test_long_cache_offsets_pass_31_bits(cuda):
    """A cache of more than 2^31 elements: the last of its heads against a call that sees that head alone."""
    import torch
    from moat_b200.tree import tree_attention
    Lmax, d = 140000, 128
    x = inputs(cuda, 1, 2, 1, 1, d, [0], 0, seed=13)
    big = torch.empty(2 ** 31 // (Lmax * d) + 2, Lmax, d, dtype=torch.float16, device=cuda)
    n = big.shape[0]
    kb = big.as_strided((1, 1, Lmax, d), (0, 0, d, 1), (n - 1) * Lmax * d)
    kb.normal_()
    v = torch.randn((1, 1, Lmax, d), device=cuda).half()
    whole = big.view(1, n, Lmax, d)
    q, kd, vd, masks = x["q"], x["k_draft"], x["v_draft"], x["masks"]
    lens = torch.tensor([139000], dtype=torch.int32, device=cuda)
    qn = q.expand(1, 2, n, d).contiguous()
    got = tree_attention(qn, whole, v.expand(1, n, Lmax, d), lens, kd.expand(1, 2, n, d), vd.expand(1, 2, n, d), masks)
    want = tree_attention(q, kb, v, lens, kd, vd, masks)
    u = U["float16"]
    assert bool(((got[:, :, -1:] - want).abs().double() <= 4 * u * want.abs().double().clamp(min=0.05)).all())


# ---------------------------------------------------------------------------------------
# acceptance
# ---------------------------------------------------------------------------------------
def walk(tokens, parents, target):
    """Greedy acceptance of one trace on the host."""
    if tokens[0] < 0:
        return [], -1
    path = [0]
    while True:
        nxt = [i for i in range(path[-1] + 1, len(tokens))
               if parents[i] == path[-1] and tokens[i] >= 0 and tokens[i] == target[path[-1]]]
        if not nxt:
            return path, target[path[-1]]
        path.append(nxt[0])


@pytest.mark.parametrize("layers,T,Hkv,d,m", [(None, 1, 1, 64, 1), (None, 3, 2, 64, 5), (3, 4, 2, 128, 16),
                                              (2, 9, 3, 72, 64), (1, 2, 2, 33, 33)])
def test_accept(cuda, layers, T, Hkv, d, m):
    import torch
    from moat_b200.tree import accept_tree
    rng = np.random.default_rng(m)
    # few distinct tokens: long accepted paths, siblings with the same token
    tokens, target = rng.integers(0, 2, (T, m)), rng.integers(0, 2, (T, m))
    parents = random_parents(rng, T, m)
    parents[:, m - m // 4:] = -1  # padding
    if T > 2:
        tokens[1, 0] = -7  # an idle trace
    Lmax, lead = 96, () if layers is None else (layers,)
    lens = rng.integers(0, Lmax - m, T)
    dev = dict(device=cuda)

    def i32(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(cuda)

    k, v = (torch.randn(lead + (T, Hkv, Lmax, d), **dev).half() for _ in range(2))
    kd, vd = (torch.randn(lead + (T, m, Hkv, d), **dev).half() for _ in range(2))
    scores, ds = torch.rand(lead + (T, Hkv, Lmax), **dev), torch.rand(lead + (T, Hkv, m), **dev)
    pos = torch.zeros(lead + (T, Hkv, Lmax), dtype=torch.int32, **dev)
    want = [x.clone() for x in (k, v, scores, pos)]
    got = accept_tree(i32(tokens), i32(parents), i32(target), i32(lens), i32(lens + 10), k, v, kd, vd, scores=scores,
                      draft_scores=ds, positions=pos)
    for t in range(T):
        path, nxt = walk(tokens[t], parents[t], target[t])
        n = len(path)
        assert got.path[t].tolist() == path + [-1] * (m - n)
        assert (int(got.counts[t]), int(got.next_ids[t])) == (n, nxt)
        assert (int(got.lens[t]), int(got.next_pos[t])) == (lens[t] + n, lens[t] + 10 + n)
        for j, node in enumerate(path):
            row = lens[t] + j
            want[0][..., t, :, row, :] = kd[..., t, node, :, :]
            want[1][..., t, :, row, :] = vd[..., t, node, :, :]
            want[2][..., t, :, row] = ds[..., t, :, node]
            want[3][..., t, :, row] = int(lens[t]) + 10 + j
    for a, b in zip((k, v, scores, pos), want):
        assert torch.equal(a, b)  # accepted rows copied, every other row untouched


def test_accept_without_room_keeps_the_trace(cuda):
    import torch
    from moat_b200.tree import accept_tree
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    k = torch.zeros((3, 1, 8, 64), dtype=torch.float16, device=cuda)
    kd = torch.ones((3, 2, 1, 64), dtype=torch.float16, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    v = k.clone()
    r = accept_tree(i32([[5, 6]] * 3), i32([-1, 0]), i32([[6, 9]] * 3), i32([6, 7, 8]), i32([6, 7, 8]), k, v, kd,
                    kd.clone(), dev_err=err)
    assert r.counts.tolist() == [2, 0, 0] and r.next_ids.tolist() == [9, -1, -1] and r.lens.tolist() == [8, 7, 8]
    assert int(err) == 2
    assert k[0, 0, :, 0].tolist() == [0] * 6 + [1] * 2 and not bool(k[1:].any()) and not bool(v[1:].any())


def test_accept_strided_drafts(cuda):
    import torch
    from moat_b200.tree import accept_tree
    T, m, Hkv, d = 2, 4, 2, 64
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    qkv = torch.randn((T, m, 6 * d), device=cuda).half()
    kd, vd = qkv[..., 2 * d:4 * d].view(T, m, Hkv, d), qkv[..., 4 * d:].view(T, m, Hkv, d)
    k = torch.zeros((T, 10, Hkv, d), dtype=torch.float16, device=cuda).transpose(1, 2)
    v = torch.zeros((T, Hkv, 10, d + 1), dtype=torch.float16, device=cuda)[..., :d]
    accept_tree(i32([[1, 2, 3, 4]] * T), i32([-1, 0, 1, 2]), i32([[2, 3, 0, 0]] * T), i32([1, 5]), i32([1, 5]), k, v,
                kd, vd)
    for t, n in enumerate([1, 5]):
        for j in range(3):
            assert torch.equal(k[t, :, n + j], kd[t, j]) and torch.equal(v[t, :, n + j], vd[t, j])
        assert not bool(k[t, :, n + 3:].any()) and not bool(v[t, :, :n].any())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_rope_of_a_tree(cuda, dtype):
    import torch
    from moat_b200._lib import lib, stream_of
    from moat_b200.decode import rope_table
    T, m, H, Hkv, dh = 2, 5, 4, 2, 64
    dt = getattr(torch, dtype)
    qkv = torch.randn((T, m, (H + 2 * Hkv) * dh), device=cuda).to(dt)
    cs = rope_table(dh, 50, 10000.0).to(cuda)
    pos = torch.tensor([3, 45], dtype=torch.int32, device=cuda)
    depth = torch.tensor([0, 1, 1, 2, 9], dtype=torch.int32, device=cuda)
    q, k = torch.zeros((T, m, H, dh), dtype=dt, device=cuda), torch.zeros((T, m, Hkv, dh), dtype=dt, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert lib().mb_tree_rope(qkv.data_ptr(), int(dt == torch.bfloat16), T, m, H, Hkv, dh, pos.data_ptr(),
                              depth.data_ptr(), 1, cs.data_ptr(), 50, q.data_ptr(), k.data_ptr(), err.data_ptr(),
                              stream_of(cuda)) == 0
    assert int(err) == 2  # trace 1's last node lies past the table: skipped
    x = qkv[..., :(H + Hkv) * dh].double().view(T, m, H + Hkv, dh // 2, 2)
    got = torch.cat([q, k], 2).double().view(T, m, H + Hkv, dh // 2, 2)
    for t in range(T):
        for i in range(m):
            p = int(pos[t] + depth[i])
            if p >= 50:
                assert not bool(got[t, i].any())
                continue
            c, s = cs[p].double().unbind(-1)
            want = torch.stack([x[t, i, ..., 0] * c - x[t, i, ..., 1] * s, x[t, i, ..., 0] * s + x[t, i, ..., 1] * c], -1)
            # products and their difference in fp32, one rounding to the element type
            bound = 1.1 * U[dtype] * want.abs() + 2.0 ** -22 * x[t, i].abs().sum(-1, keepdim=True) + 2.0 ** -24
            assert bool(((got[t, i] - want).abs() <= bound).all())


def test_refusals(cuda):
    import torch
    from moat_b200.tree import accept_tree, tree_attention
    x = inputs(cuda, 2, 4, 8, 2, 64, [5, 9], 16, seed=1)

    def refuse(error=ValueError, **change):
        with pytest.raises(error):
            tree_attention(**{**x, **change})

    refuse(TypeError, q=x["q"].cpu().numpy())
    refuse(q=x["q"].cpu())
    refuse(q=x["q"].float())
    refuse(q=x["q"].bfloat16())  # another dtype than the caches
    refuse(q=x["q"][:, :, :7])  # 7 heads over 2
    refuse(q=x["q"][0])
    refuse(q=x["q"].transpose(2, 3).contiguous().transpose(2, 3))  # head dim not contiguous
    refuse(v_cache=x["v_cache"][:, :, :8])
    refuse(k_draft=x["k_draft"][:, :3])
    refuse(lens=x["lens"].long())
    refuse(lens=x["lens"][:1])
    refuse(masks=x["masks"].int())
    refuse(masks=x["masks"][:, :3])
    refuse(out=x["q"][:1])
    refuse(scale=float("inf"))
    refuse(scores_out=torch.zeros((2, 2, 16), device=cuda))
    refuse(scores=torch.zeros((2, 2, 15), device=cuda))
    refuse(scores=torch.zeros((2, 2, 16), device=cuda).half())
    wide = inputs(cuda, 1, 1, 1, 1, 264, [5], 16, seed=1)
    with pytest.raises(ValueError):
        tree_attention(**wide)
    i = torch.zeros((2, 4), dtype=torch.int32, device=cuda)
    n = x["lens"]
    args = dict(tokens=i, parents=i, target=i, lens=n, next_pos=n, k_cache=x["k_cache"], v_cache=x["v_cache"],
                k_draft=x["k_draft"], v_draft=x["v_draft"])
    for change in (dict(tokens=i.long()), dict(parents=i[:, :3]), dict(lens=n[:1]), dict(k_draft=x["k_draft"][:1]),
                   dict(v_cache=x["v_cache"].float()), dict(k_cache=x["k_cache"][0]),
                   dict(scores=torch.zeros((2, 2, 16), device=cuda)),
                   dict(positions=torch.zeros((2, 2, 16), device=cuda)), dict(target=i.cpu())):
        with pytest.raises(ValueError):
            accept_tree(**{**args, **change})
