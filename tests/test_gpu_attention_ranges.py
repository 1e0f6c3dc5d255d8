"""Scored attention at the ends of what its arguments may be, against the formula in 64 bits:
caps far above and far below the scores, and values near the largest number.

Tolerances are those of test_gpu_attention_scores.py but for a capped score, whose error is
relative to the score here and not to the cap.  u = 2^-24, x = s / cap before the cap:
  - |x| < 1/4: s times a polynomial in x^2, 1 to 0.98: the product with the scale and the
    scale's own rounding 2 u, x^2 3 u times a slope of at most x^2 / 3 < 0.03, five steps of the
    polynomial of which all but the last count for at most x^2 (2 u together), the product u,
    and the terms left out 2^-26: under 6 u |s|;
  - above: cap (1 - 2 r), r = 1 / (1 + e^2x): the exponent off by 3 u |2 x| and the
    exponential by 2 u move r by r (1 - r) (6 |x| + 2) u, the sum and the reciprocal by 3 u r;
    2 r takes its part of cap twice over, the last step rounds once: at most cap u (0.5 (6 / 4 +
    2) + 6 + 1) = 8.8 cap u, where |s| >= cap tanh(1/4) = 0.244 cap: 36 u |s|.  (Beyond |x| = 1/4
    r (1 - r) |x| falls: at 1 it is 0.105, 1.7 u; at 3 under 0.01.)
The bound taken is 40 u |s|.  The any-size kernels' cap tanhf(x), tanhf within 2 steps, keeps it too."""

import math

import pytest
import torch

import pxs
from test_gpu_attention_scores import B, U, alibi, bounds, check, formula, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def capped(q, k, v, q_len, k_len, heads, kv, d, scale, cap, slopes=None, causal=False):
    """-> (values, tolerance) [rows, heads * d] in 64 bits on the CPU."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    out = torch.zeros((sum(q_len), heads, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    q0 = k0 = 0
    for nq, nk in zip(q_len, k_len):
        away = torch.arange(nk - nq, nk)[:, None] - torch.arange(nk)[None, :]
        for h in range(heads):
            g = h // (heads // kv)
            qs = q[q0:q0 + nq, h * d:(h + 1) * d]
            ks, vs = (t[k0:k0 + nk, g * d:(g + 1) * d] for t in (k, v))
            s = cap * torch.tanh(qs @ ks.T * scale / cap)
            e = (qs.abs() @ ks.abs().T) * scale * (d + 3) + 40.0 * s.abs()
            if slopes is not None:
                bias = float(slopes[h]) * away.abs().double()
                s, e = s - bias, e + 4.0 * bias
            e = U * (e + 4.0 * s.abs())
            if causal:
                s = s.masked_fill(away < 0, -math.inf)
            p = torch.exp(s - s.amax(1, keepdim=True))
            total = p.sum(1, keepdim=True)
            o, size, pe = p @ vs / total, p @ vs.abs() / total, p * e
            out[q0:q0 + nq, h] = o
            tol[q0:q0 + nq, h] = (pe @ vs.abs() + pe.sum(1, keepdim=True) * o.abs()) / total + (nk + 16) * U * size
        q0, k0 = q0 + nq, k0 + nk
    return out.flatten(1), tol.flatten(1)


def rounded(want, tol, q, k, v):
    """The tolerance with the roundings of bf16 weights (at most 2 b of the largest value) and outputs."""
    if q.dtype == torch.float32:
        return tol + 1e-37
    tol = tol + 2 * B * float(v.abs().max())
    return tol + B * (want.abs() + tol) + 1e-37


LENGTHS = {"prompts": ([300, 129], [300, 411]), "new tokens": ([1, 1, 3], [3000, 17, 640])}


@pytest.mark.parametrize("cap", [300.0, 1e4, 1e6, 1e8, 1e30, 3e38])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 80), (torch.bfloat16, 100),
                                     (torch.float32, 64), (torch.float32, 200)])
def test_caps_above_the_scores(px, dtype, d, lengths, cap):
    """Scores of a few units under any cap, as if there were none where it is far above; and scores
    about the cap."""
    q_len, k_len = LENGTHS[lengths]
    for bias, causal, about in ((False, False, False), (True, True, False), (True, False, False), (False, True, True)):
        if about and cap > 1e6:
            continue
        gain = 0.8 * math.sqrt(cap) if about else 2.0
        print(f"[caps] {lengths} d={d} {dtype} cap={cap} bias={bias} causal={causal} gain={gain}", flush=True)
        q, k, v = inputs(q_len, k_len, 4, 2, d, dtype, 61, gain)
        slopes, scale = alibi(4) if bias else None, 1.0 / math.sqrt(d)
        o = px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(k_len), 4, 2, d, scale, cap=cap, slopes=slopes,
                                       causal=causal)
        want, tol = capped(q, k, v, q_len, k_len, 4, 2, d, scale, cap, slopes, causal)
        check(o, want, rounded(want, tol, q, k, v), f"cap {cap}")


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("d", [64, 80, 128])
def test_caps_about_the_change_of_form(px, d, lengths):
    """The largest cap of one form, and the next number, which takes the other: both near the formula."""
    q_len, k_len = LENGTHS[lengths]
    q, k, v = inputs(q_len, k_len, 4, 2, d, torch.bfloat16, 62)
    for cap in (256.0, 256.0 * (1.0 + 2.0 ** -23)):
        o = px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(k_len), 4, 2, d, 0.2, cap=cap, causal=True)
        want, tol = formula(q, k, v, q_len, k_len, 4, 2, d, 0.2, cap, None, True)
        check(o, want, tol, f"cap {cap}")


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_caps_far_below_the_scores(px, dtype, lengths):
    """Caps so small that every score is next to nothing: the mean of the values, also where a product
    is zero and its multiplier past what fp32 holds."""
    q_len, k_len = LENGTHS[lengths]
    q, k, v = inputs(q_len, k_len, 4, 2, 64, dtype, 63)
    q[0] = 0.0
    for cap in (1e-20, 1e-39):
        o = px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(k_len), 4, 2, 64, 0.125, cap=cap)
        want, tol = formula(q, k, v, q_len, k_len, 4, 2, 64, 0.125, 1e-20)
        check(o, want, tol, f"cap {cap}")


def test_small_scale_under_a_large_cap(px):
    """A scale that its cap divides to a subnormal number, or to nothing, still scales the scores."""
    for dtype, d in ((torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 200)):
        for q_len, k_len in LENGTHS.values():
            q, k, v = inputs(q_len, k_len, 2, 2, d, dtype, 64)
            for scale, cap in ((1e-4, 3e38), (1e-10, 3e38)):
                big = (q.float() * (0.1 / scale)).to(dtype)
                o = px.varlen_attention_scores(big, k, v, bounds(q_len), bounds(k_len), 2, 2, d, scale, cap=cap)
                want, tol = formula(big, k, v, q_len, k_len, 2, 2, d, scale)
                check(o, want, tol, f"scale {scale}")


def heads_of(px, q, k, v, q_len, k_len, heads, kv, d, scale, sample, what, cap=0.0, bias=False, causal=False, prefix=None):
    """The call, and the sampled heads of its output against the formula."""
    slopes = alibi(heads) if bias else None
    o = px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(k_len), heads, kv, d, scale, cap=cap, slopes=slopes,
                                   causal=causal, prefix=None if prefix is None else torch.tensor(prefix, device="cuda"))
    for h in sample:
        cols, kv_cols = slice(h * d, (h + 1) * d), slice(h // (heads // kv) * d, (h // (heads // kv) + 1) * d)
        want, tol = formula(q[:, cols], k[:, kv_cols], v[:, kv_cols], q_len, k_len, 1, 1, d, scale, cap,
                            None if slopes is None else slopes[h:h + 1], causal, prefix)
        check(o[:, cols], want, tol, f"{what}, head {h}")


@pytest.mark.parametrize("heads", [2, 40])  # the keys split over workgroups, and walked by one
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("mode", [dict(), dict(causal=True), dict(causal=True, bias=True), dict(cap=100.0)])
def test_large_values_under_rising_scores(px, d, heads, mode):
    """Values near the largest number, and scores that rise by e^25 along the walk from the last key to the
    first: no weight may carry the sums past what fp32 holds where the result is well within."""
    n = 900
    gen = torch.Generator("cuda").manual_seed(65)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    q, k = 0.02 * rand(n, heads, d), rand(n, heads, d)
    q[:, :, 0], k[:, :, 0] = 1.0, 0.0
    for at, score in ((10, 45.0), (300, 25.0), (480, 25.0), (700, 20.0)):
        k[at, :, 0] = score
    q, k = (t.reshape(n, heads * d).bfloat16() for t in (q, k))
    for size in (1e30, 1e36):
        v = (size * rand(n, heads * d)).bfloat16()
        print(f"[scores] large values d={d} heads={heads} {mode} {size}", flush=True)
        heads_of(px, q, k, v, [n], [n], heads, heads, d, 1.0, [0, heads - 1], f"values of {size}", **mode)
