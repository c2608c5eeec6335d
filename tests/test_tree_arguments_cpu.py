"""More argument checks of drafted decoding's C entry points: they fail before any CUDA call, so
the addresses are never looked at."""

import ctypes
import struct

import pytest

from moat_b200 import _lib

FAKE, OTHER, ODD = 0x10000, 0x20000, 0x30002


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def attention(L, err=0, strides=(128,) * 18, T=1, m=4, H=8, Hkv=2, Lmax=64, nbytes=1 << 30):
    """mb_tree_attn_args; without a workspace, a call that passes the checks before it ends with -3."""
    return L.mb_tree_attn(struct.pack("@13PN18q8if", *[FAKE] * 8, 0, 0, 0, FAKE, err, nbytes, *strides, 0, 0, T, m, H,
                                      Hkv, Lmax, 128, 0.1), None)


def accept(L, err=0, strides=(128,) * 16, layers=1, T=1, Hkv=2, Lmax=64):
    return L.mb_tree_accept(struct.pack("@18P16q7i", *[FAKE] * 9, 0, 0, 0, FAKE, FAKE, FAKE, OTHER, OTHER, err, *strides,
                                        0, layers, T, 4, Hkv, Lmax, 128), None)


def test_the_error_word_is_aligned(L):
    assert attention(L, err=ODD) == -5
    assert accept(L, err=ODD) == -5
    fake = ctypes.c_void_p(FAKE)
    assert L.mb_tree_rope(fake, 0, 1, 4, 8, 2, 128, fake, fake, 0, fake, 64, fake, fake, ctypes.c_void_p(ODD), None) == -5


def evict(L, strides):
    return L.mb_cache_evict(struct.pack("@10PN8q8i", *[FAKE] * 4, OTHER, OTHER, FAKE, FAKE, OTHER, 0, 0, *strides, 2, 2,
                                        2, 64, 128, 32, 8, 4), None)


def test_broadcast_strides_of_what_is_written(L):
    """0 along an axis of more than one element."""
    def zero(at, n):
        return [0 if u == at else 128 for u in range(n)]
    for u in range(15, 18):
        assert attention(L, strides=zero(u, 18), T=2, nbytes=0) == -2
    assert attention(L, strides=zero(15, 18), nbytes=0) == -3  # T = 1: the stride is never used
    for u in range(15):
        assert attention(L, strides=zero(u, 18), T=2, nbytes=0) == -3  # inputs may be broadcast
    for u in range(8):
        assert accept(L, strides=zero(u, 16), layers=2, T=2) == -2
        assert evict(L, zero(u, 8)) == -2
    assert evict(L, [128] * 8) == -3


def test_the_output_in_the_queries_place_with_scores(L):
    def call(q, scores):
        return L.mb_tree_attn(struct.pack("@13PN18q8if", q, *[OTHER] * 6, FAKE, 0, scores, scores, 0, 0, 0, *[128] * 18,
                                          0, 0, 1, 4, 8, 2, 64, 128, 0.1), None)
    assert call(FAKE, OTHER) == -2
    assert call(FAKE, 0) == -3 and call(OTHER, OTHER) == -3


def test_weights_without_a_cache_need_only_the_drafts(L):
    def call(Lmax, scores_out, draft, cache=0, m=4):
        return L.mb_tree_attn(struct.pack("@13PN18q8if", FAKE, cache, cache, FAKE, FAKE, FAKE, FAKE, OTHER, 0, scores_out,
                                          draft, 0, 0, 0, *[128] * 18, 0, 0, 1, m, 8, 2, Lmax, 128, 0.1), None)
    assert call(0, 0, FAKE) == -3 and call(0, FAKE, FAKE) == -3 and call(0, 0, 0) == -3
    assert call(0, FAKE, 0) == -1  # nowhere to put the drafts' sums
    assert call(1, 0, FAKE, cache=FAKE) == -1  # nor the rows'


def test_masks_of_missing_drafts():
    """A node without a token, and what hangs on it, is padding; the others keep their ancestors."""
    import types

    import torch
    from moat_b200.speculative import TreeDecoder
    from moat_b200.tree import tree_masks
    parents = [-1, 0, 0, 1, 2, 3] + list(range(5, 63))
    masks = torch.from_numpy(tree_masks(parents))
    tokens = torch.zeros((4, 64), dtype=torch.int32)
    tokens[1, 1] = -1
    tokens[2, 63] = -7
    tokens[3, 0] = -1
    s = types.SimpleNamespace(tokens=tokens, masks=masks, nodes=torch.arange(64))
    got = TreeDecoder._drafted_masks(None, s)
    assert got.is_contiguous() and got.dtype == torch.int64
    assert torch.equal(got[0], masks) and torch.equal(got[2, :63], masks[:63]) and int(got[2, 63]) == 0
    assert [i for i in range(64) if got[1, i] != 0] == [0, 2, 4]
    assert int(got[1, 4]) == 0b10101 and not bool(got[3].any())


def test_device_error_words_are_spelled_out():
    _lib.check_device(0, "a step")
    for word, text in ((1, "wait"), (2, "index"), (3, "wait.*index"), (4, "finite"), (1 << 20, "unknown")):
        with pytest.raises(_lib.MoatError, match=text):
            _lib.check_device(word, "a step")
