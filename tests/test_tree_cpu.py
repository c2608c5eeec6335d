"""Host logic of drafted decoding: tree masks and depths, workspace sizes, and the
argument checks of the C entry points (they fail before any CUDA call)."""

import ctypes
import struct

import numpy as np
import pytest

from moat_b200 import _lib
from moat_b200.tree import tree_depths, tree_masks


def test_masks_and_depths_of_a_small_tree():
    #      0
    #    1   2
    #    4   3     node 5: its parent is padding, node 6: parent after itself
    par = [-1, 0, 0, 2, 1, 7, 6, -1]
    np.testing.assert_array_equal(tree_masks(par), [0b1, 0b11, 0b101, 0b1101, 0b10011, 0, 0, 0])
    np.testing.assert_array_equal(tree_depths(par), [0, 1, 1, 2, 2, 0, 0, 0])


def test_descendants_of_padding_are_padding():
    np.testing.assert_array_equal(tree_masks([-1, -1, 1, 0]), [1, 0, 0, 0b1001])


def test_full_width_chain_uses_all_64_bits():
    par = np.arange(64) - 1
    masks = tree_masks(np.stack([par, par])).view(np.uint64)
    assert masks.shape == (2, 64)
    for i in range(64):
        assert int(masks[1, i]) == (1 << (i + 1)) - 1
    np.testing.assert_array_equal(tree_depths(par), np.arange(64))


@pytest.mark.parametrize("seed", range(4))
def test_masks_match_a_walk_to_the_root(seed):
    rng = np.random.default_rng(seed)
    par = np.array([[-1] + [int(rng.integers(-1, i)) for i in range(1, 40)] for _ in range(3)])
    masks, depths = tree_masks(par).view(np.uint64), tree_depths(par)
    for t in range(3):
        for i in range(40):
            seen, j = [i], i
            while j > 0 and par[t, j] >= 0:
                j = par[t, j]
                seen.append(j)
            want = sum(1 << s for s in seen) if j == 0 else 0
            assert int(masks[t, i]) == want
            assert depths[t, i] == (len(seen) - 1 if j == 0 else 0)


@pytest.mark.parametrize("m", [0, 65])
def test_tree_sizes_are_refused(m):
    with pytest.raises(ValueError):
        tree_masks([-1] * m)


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def test_workspace_sizes(L):
    assert L.mb_tree_attn_workspace_size(2, 8, 16, 4, 1024, 128, 0) > 0
    for bad in [(0, 8, 16, 4, 1024, 128), (2, 65, 16, 4, 1024, 128), (2, 8, 15, 4, 1024, 128),
                (2, 8, 16, 4, 1024, 257), (2, 8, 16, 4, -1, 128)]:
        assert L.mb_tree_attn_workspace_size(*bad, 1) == 0
    assert L.mb_cache_evict_workspace_size(1, 1, 4, 320, 256) >= 4 * 2 * 64 * 4
    assert L.mb_cache_evict_workspace_size(1, 1, 4, 320, 0) == 0


FAKE, OTHER = 0x10000, 0x20000  # never dereferenced: validation fails first
# the C structs mb_tree_attn_args, mb_tree_accept_args and mb_cache_evict_args
_AttnArgs = struct.Struct("@13PN18q8if")
_AcceptArgs = struct.Struct("@18P16q7i")
_Args = struct.Struct("@10PN8q8i")


def test_attention_entry_checks_its_arguments(L):
    def attn(q=FAKE, k=FAKE, masks=FAKE, bf16=0, T=1, m=4, H=8, Hkv=2, Lmax=64, d=128, scale=0.1, scores=0,
             scores_out=0, draft=0, ws=FAKE, nbytes=1 << 30):
        return L.mb_tree_attn(_AttnArgs.pack(q, k, FAKE, FAKE, FAKE, FAKE, masks, FAKE, scores, scores_out, draft, ws, 0,
                                             nbytes, *[128] * 18, 0, bf16, T, m, H, Hkv, Lmax, d, scale), None)
    assert L.mb_tree_attn(None, None) == -1
    assert attn(q=0) == -1
    assert attn(k=0) == -1
    assert attn(masks=0) == -1
    assert attn(scores_out=FAKE) == -1  # draft_scores missing
    assert attn(scores=FAKE) == -1  # nowhere to put the sums
    assert attn(m=0) == -2 and attn(m=65) == -2
    assert attn(H=7) == -2 and attn(Hkv=0) == -2
    assert attn(d=257) == -2 and attn(T=0) == -2 and attn(Lmax=-1) == -2
    assert attn(scale=float("inf")) == -2 and attn(scale=float("nan")) == -2
    assert attn(bf16=2) == -2
    assert attn(ws=0) == -3 and attn(nbytes=16) == -3
    assert attn(q=0x10001) == -5
    assert attn(masks=0x10004) == -5


def test_accept_entry_checks_its_arguments(L):
    def accept(tokens=FAKE, lens=FAKE, layers=1, T=1, m=4, Hkv=2, Lmax=64, d=128, scores=0, draft=0, lens_out=OTHER,
               pos_out=OTHER):
        return L.mb_tree_accept(_AcceptArgs.pack(tokens, FAKE, FAKE, lens, FAKE, FAKE, FAKE, FAKE, FAKE, scores, draft, 0,
                                                 FAKE, FAKE, FAKE, lens_out, pos_out, 0, *[128] * 16, 0, layers, T, m,
                                                 Hkv, Lmax, d), None)
    assert L.mb_tree_accept(None, None) == -1
    assert accept(tokens=0) == -1
    assert accept(scores=FAKE) == -1  # draft_scores missing
    assert accept(m=65) == -2 and accept(T=0) == -2 and accept(layers=0) == -2 and accept(Lmax=0) == -2
    assert accept(lens_out=FAKE) == -2  # in place: another CTA may still read the old length
    assert accept(pos_out=FAKE) == -2
    assert accept(layers=70000) == -6 and accept(Hkv=70000) == -6


def test_rope_and_evict_entries_check_their_arguments(L):
    fake = ctypes.c_void_p(FAKE)
    assert L.mb_tree_rope(None, 0, 1, 4, 8, 2, 128, fake, fake, 0, fake, 64, fake, fake, None, None) == -1
    assert L.mb_tree_rope(fake, 0, 1, 4, 8, 2, 127, fake, fake, 0, fake, 64, fake, fake, None, None) == -2
    assert L.mb_tree_rope(fake, 0, 1, 65, 8, 2, 128, fake, fake, 0, fake, 64, fake, fake, None, None) == -2
    assert L.mb_tree_rope(fake, 0, 1, 4, 8, 2, 128, fake, fake, 0, ctypes.c_void_p(0x10004), 64, fake, fake, None,
                          None) == -5

    def evict(k=FAKE, so=OTHER, po=OTHER, lens_out=OTHER, budget=32, recent=8, sinks=4, ws=FAKE, nbytes=1 << 30, Lmax=64):
        return L.mb_cache_evict(_Args.pack(k, FAKE, FAKE, FAKE, so, po, FAKE, FAKE, lens_out, ws, nbytes, *[128] * 8, 1, 1,
                                           2, Lmax, 128, budget, recent, sinks), None)
    assert L.mb_cache_evict(None, None) == -1
    assert evict(k=0) == -1
    assert evict(budget=0) == -2 and evict(recent=-1) == -2 and evict(sinks=-1) == -2
    assert evict(budget=11) == -2  # cannot hold the recent rows and the sinks
    assert evict(lens_out=FAKE) == -2
    assert evict(so=FAKE) == -2  # scores in place, positions not
    assert evict(Lmax=0) == -2
    assert evict(Lmax=1 << 20) == -6  # more rows than a cluster's shared memory ranks
    assert evict(ws=0) == -3 and evict(nbytes=16) == -3


def test_argument_structs_match_the_header():
    """The packed formats have the size that the compiler gives the structs of the header."""
    import subprocess
    import tempfile
    src = ('#include <stdio.h>\n#include "moat_b200.h"\nint main(void) { printf("%zu %zu %zu %zu", '
           'sizeof(mb_tree_attn_args), sizeof(mb_tree_accept_args), sizeof(mb_cache_evict_args), '
           'offsetof(mb_tree_attn_args, scale)); return 0; }\n')
    with tempfile.TemporaryDirectory() as tmp:
        c, exe = f"{tmp}/s.c", f"{tmp}/s"
        with open(c, "w") as f:
            f.write(src)
        root = __file__.rsplit("/", 2)[0]
        subprocess.run(["gcc", "-I", f"{root}/include", c, "-o", exe], check=True)
        sizes = [int(x) for x in subprocess.run([exe], capture_output=True, check=True, text=True).stdout.split()]
    pad = [-(-s.size // 8) * 8 for s in (_AttnArgs, _AcceptArgs, _Args)]
    assert sizes[:3] == pad and sizes[3] == _AttnArgs.size - 4


def test_lookup_draft():
    from moat_b200.speculative import lookup_draft
    assert lookup_draft([5, 1, 2, 3, 4, 1, 2], 4) == [3, 4, 1]  # after the earlier "1 2"
    assert lookup_draft([7, 8, 9, 8], 3) == [9, 8]  # after the earlier "8"
    assert lookup_draft([1, 2, 3], 5) == [-1] * 4
    assert lookup_draft([4, 4], 4) == [4, -1, -1]
    assert lookup_draft([], 1) == []
