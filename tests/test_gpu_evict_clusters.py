"""Eviction of caches that a cluster of CTAs ranks: every size launches, whatever ran before it
in the process, and gives what the host implementation gives."""

import os
import subprocess
import sys

import pytest

from test_gpu_evict import run

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
# rows that make 7,936 per CTA of a cluster of 2, 4 and 8 (the largest and the smallest)
SIZES = [15617, 15872, 31233, 31744, 62465, 63488]


@pytest.mark.parametrize("Lmax", SIZES)
def test_sizes_launch_first_in_a_process(cuda, Lmax):
    """A kernel's limit of shared memory stays raised once it has been, so each size has a process of its own."""
    code = f"""
import sys
sys.path[:0] = [{HERE!r}, {os.path.dirname(HERE)!r}]
import torch
from test_gpu_evict import run
run(torch.device("cuda:0"), None, 1, 2, {Lmax}, 16, [{Lmax - 3}], 5000, 64, 4, seed=1)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T,Hkv,Lmax,d,lens,budget,recent,sinks", [
    (1, 2, 15872, 64, [15872], 7000, 100, 4),  # clusters of 2
    (3, 12, 12001, 72, [12000, 6001, 3], 6000, 50, 0),
    (1, 2, 31700, 33, [31699], 31000, 0, 0),  # of 4
    (2, 4, 20000, 64, [20000, 19999], 300, 200, 100),
    (1, 1, 63001, 64, [63000], 40000, 300, 4),  # of 8
])
def test_clusters(cuda, T, Hkv, Lmax, d, lens, budget, recent, sinks, in_place):
    run(cuda, None, T, Hkv, Lmax, d, lens, budget, recent, sinks, in_place=in_place, seed=Lmax)


def test_the_most_rows(cuda):
    """786,432 rows are what a cluster of 16 ranks; one more is refused."""
    from moat_b200._lib import MoatError
    n = 786432
    run(cuda, None, 1, 1, n, 8, [n], 300000, 1000, 4)
    with pytest.raises(MoatError):
        run(cuda, None, 1, 1, n + 1, 8, [n], 300000, 1000, 4)
