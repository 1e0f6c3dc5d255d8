"""Tree attention (pxs_tree_attention) of values near the largest number: a mean of them is one, whatever
the number of keys, and however the call is cut.  Against the formula in 64 bits, with the tolerances of
test_gpu_attention_tree.py."""

import math

import pytest
import torch

import pxs
from test_gpu_attention_scores import check
from test_gpu_attention_tree import Batch
from test_gpu_attention_tree_paths import plan, want

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
KINDS = [(F32, 64), (F32, 128), (F32, 256), (F32, 99), (F32, 200), (BF16, 64), (BF16, 128), (BF16, 40), (BF16, 96), (BF16, 99),
         (BF16, 200), (BF16, 256)]


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def sized(b, value):
    """Every value `value`, of one sign or as it was drawn."""
    for t in (b.vc, b.v):
        t.copy_((torch.ones_like(t) if value > 0 else torch.sign(t)) * abs(value))


@pytest.mark.parametrize("gain", [0.0, 0.5, 4.0])
@pytest.mark.parametrize("value", [1e35, 3e38, -3e38])
@pytest.mark.parametrize("dtype,d", KINDS)
def test_means_of_large_values(px, dtype, d, value, gain):
    """Over 4,096 keys and few, in one chunk and many; scores all alike, near one another and far apart."""
    print(f"[tree sizes] {dtype} d={d} {value} {gain}", flush=True)
    for q_len, k_len, heads, kv in (([5, 40], [4096, 17], 4, 2), ([3], [40000], 8, 8), ([70], [0], 2, 1), ([600, 1], [3000, 90], 8, 2)):
        b = Batch(q_len, k_len, heads, kv, d, dtype, 41, gain=gain)
        sized(b, value)
        check(b.run(px), *want(b), f"{q_len} over {k_len}")


@pytest.mark.parametrize("dtype,d", KINDS)
def test_one_chunk_of_large_values_among_others(px, dtype, d):
    """Values of ordinary size, of 2^116 and of 2^127 in stretches of their own, cut into many chunks."""
    b = Batch([9, 2], [9000, 2000], 8, 8, d, dtype, 42, gain=0.5)
    assert plan(dtype, [9, 2], [9000, 2000], 8, 8, d)["chunk"] < 600
    b.vc[b.start[0] + 1000:b.start[0] + 3000] *= 2.0 ** 116
    b.vc[b.start[0] + 5000:b.start[0] + 5700] = 2.0 ** 127
    b.vc[b.start[1] + 900:b.start[1] + 901] = -(2.0 ** 127)
    check(b.run(px), *want(b), "stretches")


@pytest.mark.parametrize("dtype,d", KINDS)
def test_large_values_beside_hidden_nan(px, dtype, d):
    """The rows that are taken alone for a token that is not finite hold large values too."""
    b = Batch([40, 6], [700, 4096], 4, 2, d, dtype, 43, gain=0.5)
    sized(b, 3e38)
    expected, tol = want(b)
    b.parents[0] = [-1] * 40
    b.t_parents[:40] = -1
    expected, tol = want(b)
    b.v[39], b.v[12] = math.nan, math.inf
    got = b.run(px)
    rows = [r for r in range(b.rows) if r not in (12, 39)]
    check(got[rows], expected[rows], tol[rows], "beside NaN")
