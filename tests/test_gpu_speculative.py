"""Drafted decoding end to end: the tokens are greedy decoding's whatever is drafted.

Every emitted token is checked against the CPU decoder oracle (fp32, exact softmax, the
same dequantized weights) fed that trace's own tokens: the logits of each accepted node
agree with it to the decoder tests' 2e-2 (fp16 GEMM inputs and outputs through two layers),
and the token is the argmax of the step's own logits.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=256, heads=2, head_dim=128, ffn=512, max_len=96)


def make(cuda, vocab=1000, seed=3, N=3, **kw):
    from moat_b200.decode import DecoderConfig, Int4Decoder
    from moat_b200.speculative import TreeDecoder
    dec = Int4Decoder(DecoderConfig(vocab=vocab, **CFG), N, device=cuda, seed=seed)
    return dec, TreeDecoder(dec, **kw)


def oracle_logits(dec, tokens):
    """fp32 logits after every token of one trace."""
    import torch
    from oracle.decoder import CpuDecoder
    d = dec.dense_weights()
    cpu = CpuDecoder(d["layers"], d["final_norm"], d["lm_head"], d["embed"], d["cis"], dec.cfg.heads, 1, len(tokens),
                     eps=dec.cfg.eps)
    with torch.no_grad():
        return torch.cat([cpu.step([tok]) for tok in tokens]).numpy()


def prompt(cuda, N, P, vocab, seed=5):
    import torch
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randint(0, vocab, (N, P), generator=g, device=cuda, dtype=torch.int32)


def run_checked(dec, spec, steps, draft):
    """generate(), recording every step's logits of the accepted nodes by position."""
    seen = [{} for _ in range(spec.N)]
    accept = spec._accept

    def spy(s, target):
        first = spec.next_pos.tolist()
        r = accept(s, target)
        if target is spec.target:
            lg = spec.logits.view(spec.N, spec.m, -1).float().cpu().numpy()
            for n, path in enumerate(r.path.tolist()):
                for j, node in enumerate(i for i in path if i >= 0):
                    seen[n][first[n] + j] = lg[n, node]
        return r

    spec._accept = spy
    out = spec.generate(steps, draft)
    del spec._accept
    for n, hist in enumerate(spec.history):
        want = oracle_logits(dec, hist[:-1])
        assert sorted(seen[n]) == list(range(len(hist) - 1 - len(out[n]), len(hist) - 1))
        for pos, got in seen[n].items():
            np.testing.assert_allclose(got, want[pos], rtol=2e-2, atol=2e-2)
            assert hist[pos + 1] == int(np.argmax(got))
    assert int(spec.dev_err) == 0
    return out


@pytest.mark.parametrize("vocab", [1000, 1152])
@pytest.mark.parametrize("parents", [[-1], [-1, 0, 1, 2, 3], [-1, 0, 0, 1, 1, 2, 3, 3]])
def test_any_draft_gives_greedy_tokens(cuda, parents, vocab):
    rng = np.random.default_rng(1)
    dec, spec = make(cuda, vocab, parents=parents)
    spec.prefill(prompt(cuda, 3, 11, vocab), chunk=4)
    out = run_checked(dec, spec, 5, lambda hist, m: rng.integers(-1, vocab, m - 1).tolist())
    assert all(len(tokens) >= 5 for tokens in out)


def test_a_right_draft_is_accepted_whole(cuda):
    """The first run's tokens as the second run's drafts, in a chain and on a branch."""
    _, plain = make(cuda, parents=[-1])
    plain.prefill(prompt(cuda, 3, 9, 1000))
    truth = plain.generate(13)
    dec, spec = make(cuda, parents=[-1, 0, 0, 2, 3])  # node 1 is a dead end, 2 - 3 - 4 the path
    spec.prefill(prompt(cuda, 3, 9, 1000))
    told = {tuple(h[-9:]): t for h, t in zip([list(h) for h in spec.history], truth)}

    def draft(hist, m):
        done = len(hist) - 9
        ahead = told[tuple(hist[:9])][done:done + 3]
        return [999 - ahead[0]] + ahead + [-1] * (3 - len(ahead)) if ahead else [-1] * (m - 1)

    got = run_checked(dec, spec, 3, draft)
    for a, b in zip(got, truth):
        assert len(a) == 12 and a == b[:12]


def test_prefill_in_chunks_matches_token_by_token(cuda):
    import torch
    ids = prompt(cuda, 3, 23, 1000)
    caches = []
    for chunk in (1, 7, 32):
        dec, spec = make(cuda, parents=[-1, 0])
        spec.prefill(ids, chunk=chunk)
        assert spec.lens.tolist() == [22] * 3 and spec.ids.tolist() == ids[:, -1].tolist()
        caches.append((spec.k_cache[..., :22, :].float(), spec.v_cache[..., :22, :].float()))
    for other in caches[1:]:
        for a, b in zip(caches[0], other):
            torch.testing.assert_close(a, b, rtol=2e-2, atol=2e-2)


def test_long_run_in_a_small_cache(cuda):
    """A budget of 40 rows: lengths stay within the capacity, positions stay unique, the recent
    rows and the sinks are there, and the scores are the weight the rows drew."""
    import torch
    dec, spec = make(cuda, parents=[-1, 0, 1, 0], capacity=56, budget=40, recent=12, sinks=2, max_positions=400)
    spec.prefill(prompt(cuda, 3, 30, 1000), chunk=8)
    out = spec.generate(70)
    assert all(len(t) >= 70 for t in out) and int(spec.dev_err) == 0
    lens, nxt = spec.lens.tolist(), spec.next_pos.tolist()
    for n in range(3):
        assert 40 <= lens[n] <= 56 and nxt[n] == 30 - 1 + len(out[n])
        for layer in range(2):
            for h in range(2):
                pos = spec.positions[layer, n, h, :lens[n]].tolist()
                assert len(set(pos)) == len(pos) and {0, 1} <= set(pos)
                assert set(range(nxt[n] - 12, nxt[n])) <= set(pos)
                assert bool((spec.scores[layer, n, h, :lens[n]] > 0).all())
    assert torch.isfinite(spec.scores).all()


def test_refusals(cuda):
    with pytest.raises(ValueError):
        make(cuda, parents=[-1] + [0] * 64)
    with pytest.raises(ValueError):
        make(cuda, parents=[-1, 0], capacity=64, budget=63)
    with pytest.raises(ValueError):
        make(cuda, parents=[-1, 0], capacity=64, budget=32, recent=40)
    dec, spec = make(cuda, parents=[-1, 0], capacity=16)
    with pytest.raises(ValueError):
        spec.step(np.zeros((3, 2), np.int32))
    with pytest.raises(ValueError):
        spec.prefill(prompt(cuda, 2, 4, 1000))
    spec.prefill(prompt(cuda, 3, 15, 1000))
    spec.generate(1, lambda h, m: [-1])
    with pytest.raises(ValueError):
        spec.generate(1, lambda h, m: [-1])  # full, and nothing may be evicted
