"""Scored attention in bf16 over many key tiles walked by one workgroup: calls with more than 256 row tiles times
key/value heads, whose keys are not split.  Most of a walk takes its weights without a maximum, two steps an
iteration, over a ring of four slots: walks of 8 to 75 tiles end it after even and odd numbers of steps, and scores
that jump by far more than 2^40 in the middle and in the last tile walked set a new base on the way.  Sampled heads are
held to the formula in 64 bits (tolerances of test_gpu_attention_scores.py, and of test_gpu_attention_ranges.py for a
cap above the scores)."""

import math

import pytest
import torch

import pxs
from test_gpu_attention_ranges import capped, heads_of, rounded
from test_gpu_attention_scores import bounds, check, formula, inputs

pytestmark = pytest.mark.gpu

MODES = [dict(), dict(causal=True), dict(cap=20.0), dict(bias=True), dict(causal=True, bias=True),
         dict(causal=True, bias=True, cap=30.0), dict(causal=True, cap=30.0, prefix=True)]


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def jumps(k, k_len, heads, d, sizes):
    """Keys that every query's first value meets with these sizes: in the middle of each segment, and among its
    first keys, the last that are walked."""
    first = 0
    for n in k_len:
        for at, size in zip((n // 2, 3), sizes):
            if n:
                k[first + min(at, n - 1)].view(heads, d)[:, 0] = size
        first += n
    return k


@pytest.mark.parametrize("mode", MODES, ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("heads,kv,d", [(40, 40, 64), (40, 20, 128), (44, 22, 96)])
@pytest.mark.parametrize("q_len,k_len", [([1000], [1000]), ([900], [2400]), ([997], [1060]), ([900, 130, 500], [900, 450, 1090])])
def test_unsplit_walks(px, q_len, k_len, heads, kv, d, mode):
    scale = 1.0 / math.sqrt(d)
    mode = dict(mode, prefix=[min(n, 333) for n in k_len]) if "prefix" in mode else mode
    for what in ("even", "jumps"):
        print(f"[walks] q={q_len} k={k_len} heads={heads}/{kv} d={d} {mode} {what}", flush=True)
        q, k, v = inputs(q_len, k_len, heads, kv, d, torch.bfloat16, 71)
        if what == "jumps":  # scores of 40 and 90, beside others of a few units
            q.view(-1, heads, d)[:, :, 0] = 8.0
            jumps(k, k_len, kv, d, (5.0 / scale, 11.25 / scale))
        heads_of(px, q, k, v, q_len, k_len, heads, kv, d, scale, (0, 17, heads - 1), what, **mode)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mode", [dict(), dict(causal=True, bias=True), dict(bias=True)], ids=lambda m: "-".join(m) or "plain")
def test_unsplit_walks_far_below_the_cap(px, d, mode):
    """The cap's other form, which has kernels of its own."""
    n, heads, scale, cap = 1060, 40, 1.0 / math.sqrt(d), 5000.0
    q, k, v = inputs([n], [n], heads, heads, d, torch.bfloat16, 72)
    q.view(n, heads, d)[:, :, 0] = 8.0
    jumps(k, [n], heads, d, (5.0 / scale, 11.25 / scale))
    slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)
    o = px.varlen_attention_scores(q, k, v, bounds([n]), bounds([n]), heads, heads, d, scale, cap=cap,
                                   slopes=slopes if "bias" in mode else None, causal="causal" in mode)
    for h in (0, 17, heads - 1):
        cols = slice(h * d, (h + 1) * d)
        want, tol = capped(q[:, cols], k[:, cols], v[:, cols], [n], [n], 1, 1, d, scale, cap,
                           slopes[h:h + 1] if "bias" in mode else None, "causal" in mode)
        check(o[:, cols], want, rounded(want, tol, q, k, v[:, cols]), f"head {h}")


def one_row(q, k, v, heads, kv, d, scale, cap):
    return formula(q[None], k, v, [1], [k.shape[0]], heads, kv, d, scale, cap, None, True)


def test_long_prompt(px):
    """A causal prompt of 5,000 tokens, and its last rows again as a call of their own: both against the formula on a
    sample of rows (whole walks of up to 157 tiles)."""
    n, heads, kv, d = 5000, 16, 8, 128
    scale = 1.0 / math.sqrt(d)
    q, k, v = inputs([n], [n], heads, kv, d, torch.bfloat16, 73)
    o = px.varlen_attention_scores(q, k, v, bounds([n]), bounds([n]), heads, kv, d, scale, cap=30.0, causal=True)
    for row in (0, 1, 31, 32, 127, 128, 2500, 4095, 4096, 4999):
        keys = row + 1
        want, tol = one_row(q[row], k[:keys], v[:keys], heads, kv, d, scale, 30.0)
        check(o[row:row + 1], want, tol, f"row {row}")
    tail = px.varlen_attention_scores(q[-700:], k, v, bounds([700]), bounds([n]), heads, kv, d, scale, cap=30.0, causal=True)
    for row in (4300, 4427, 4428, 4999):
        want, tol = one_row(q[row], k[:row + 1], v[:row + 1], heads, kv, d, scale, 30.0)
        check(tail[row - 4300:row - 4299], want, tol, f"row {row} of a chunk")
