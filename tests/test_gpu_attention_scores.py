"""Scored attention (pxs_varlen_attention_scores) against the formula in 64 bits.

Tolerances, per output o = sum p_j v_j / sum p_j, u = 2^-24 (half a step of
fp32) and b = 2^-8 (of bf16), both relative:
  - a score is off by e_j <= u ((d + 3) scale sum |q k_j| + 8 cap + 4 |s_j| + 4 slope
    |distance|): d products summed in fp32, the scale, the cap's exponential and
    reciprocal, the bias and the change to log2 units and back;
  - that moves o by at most sum p_j e_j (|v_j| + |o|) / sum p;
  - exponentials and sums of n keys in fp32: (n + 16) u sum p |v| / sum p;
  - bf16: weights are rounded, in the products and perhaps in the sum: 2 b sum p
    |v| / sum p, and so is the output: b |o|."""

import math

import numpy as np
import pytest
import torch

import pxs

pytestmark = pytest.mark.gpu
U, B = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def formula(q, k, v, q_len, k_len, heads, kv, d, scale, cap=0.0, slopes=None, causal=False, prefix=None):
    """-> (values, tolerance) [rows, heads * d] in 64 bits on the CPU.  Values of
    hidden keys are left out, whatever they hold."""
    q, k, v = (t.detach().cpu() for t in (q, k, v))
    bf16 = q.dtype == torch.bfloat16
    out = torch.zeros((sum(q_len), heads, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    q0 = k0 = 0
    for i, (nq, nk) in enumerate(zip(q_len, k_len)):
        pq, pk = torch.arange(nk - nq, nk)[:, None], torch.arange(nk)[None, :]
        seen = torch.ones((nq, nk), dtype=torch.bool)
        if causal:
            seen = pk <= pq
            if prefix is not None:
                seen = seen | (pk < prefix[i])
        for h in range(heads):
            g = h // (heads // kv)
            qs = q[q0:q0 + nq, h * d:(h + 1) * d].double()
            ks, vs = (t[k0:k0 + nk, g * d:(g + 1) * d].double() for t in (k, v))
            s = qs @ ks.T * scale
            e = (qs.abs() @ ks.abs().T) * scale * (d + 3)
            if cap > 0.0:
                s = cap * torch.tanh(s / cap)
                e = e + 8.0 * cap
            if slopes is not None:
                bias = float(slopes[h]) * (pq - pk).abs().double()
                s = s - bias
                e = e + 4.0 * bias.abs()
            e = U * (e + 4.0 * s.abs())
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(1, keepdim=True).nan_to_num(0.0, neginf=0.0)) if nk else s
            p = p.masked_fill(~seen, 0.0)
            total = p.sum(1, keepdim=True)
            total = torch.where(total == 0.0, torch.ones_like(total), total)
            never = ~seen.any(0) if nq else torch.zeros(nk, dtype=torch.bool)
            vs = vs.masked_fill(never[:, None], 0.0)
            o = torch.zeros((nq, d), dtype=torch.float64)
            if bool(torch.isfinite(vs).all()):
                o = p @ vs / total
            else:  # row by row, hidden keys left out
                for row in range(nq):
                    o[row] = (p[row, seen[row]] @ vs[seen[row]]) / total[row]
            size = p @ vs.abs().nan_to_num(0.0, posinf=0.0) / total
            pe = p * e.nan_to_num(0.0, posinf=0.0)
            t = (pe @ vs.abs().nan_to_num(0.0, posinf=0.0) + pe.sum(1, keepdim=True) * o.abs()) / total + (nk + 16) * U * size
            if bf16:
                t = t + 2 * B * size
                t = t + B * (o.abs() + t)
            out[q0:q0 + nq, h], tol[q0:q0 + nq, h] = o, t + 1e-37
        q0, k0 = q0 + nq, k0 + nk
    return out.flatten(1), tol.flatten(1)


def check(got, want, tol, what=""):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    off = (got - want).abs().nan_to_num(0.0)
    over = off - tol.nan_to_num(0.0)
    assert bool((over <= 0).all()), f"{what}: {off.flatten()[over.argmax()]:.3e} off, {tol.flatten()[over.argmax()]:.3e} allowed"


def bounds(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device="cuda")


def inputs(q_len, k_len, heads, kv, d, dtype, seed, gain=2.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    q = (gain * rand(sum(q_len), heads * d)).to(dtype)
    k, v = (gain * rand(sum(k_len), kv * d)).to(dtype), rand(sum(k_len), kv * d).to(dtype)
    return q, k, v


def alibi(heads):
    return torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)


def run_case(px, q_len, k_len, heads, kv, d, dtype, seed, cap=0.0, bias=False, causal=False, prefix=None, gain=2.0):
    print(f"[scores] q={q_len[:6]} k={k_len[:6]} segs={len(q_len)} heads={heads}/{kv} d={d} {dtype} cap={cap} "
          f"bias={bias} causal={causal} prefix={prefix}", flush=True)
    q, k, v = inputs(q_len, k_len, heads, kv, d, dtype, seed, gain)
    slopes = alibi(heads) if bias else None
    scale = 1.0 / math.sqrt(d)
    out = torch.full((sum(q_len) + 2, heads * d), 55.0, dtype=dtype, device="cuda")
    px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(k_len), heads, kv, d, scale, cap=cap, slopes=slopes,
                               causal=causal, prefix=None if prefix is None else torch.tensor(prefix, device="cuda"),
                               out=out[:sum(q_len)])
    want, tol = formula(q, k, v, q_len, k_len, heads, kv, d, scale, cap, slopes, causal, prefix)
    check(out[:sum(q_len)], want, tol, f"{q_len} over {k_len}")
    assert (out[sum(q_len):] == 55.0).all()


MODES = [dict(), dict(causal=True), dict(causal=True, cap=20.0), dict(bias=True), dict(causal=True, bias=True, cap=5.0),
         dict(cap=2.0)]
DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,d", [(4, 4, 64), (4, 2, 128), (6, 2, 64), (3, 1, 80), (2, 2, 7), (5, 1, 256), (2, 1, 200)])
def test_prompts(px, heads, kv, d, dtype, mode):
    """Ragged prompts: one token, tile ends, odd lengths, a chunk over its cache."""
    run_case(px, [1, 64, 129, 300], [1, 64, 129, 411], heads, kv, d, dtype, 1, **mode)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,d", [(16, 4, 128), (8, 8, 64), (12, 1, 64), (6, 2, 96), (64, 1, 128)])
def test_new_tokens(px, heads, kv, d, dtype, mode):
    """One or a few new tokens per sequence over caches of 1 to some thousands."""
    run_case(px, [1, 1, 1, 1, 1, 1], [3000, 1, 17, 64, 65, 777], heads, kv, d, dtype, 2, **mode)
    run_case(px, [1, 3, 5, 1], [640, 3, 1290, 127], heads, kv, d, dtype, 3, **mode)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 33])
def test_one_token_long_cache(px, d, dtype):
    """The split over a long cache: every way the last split can end."""
    for n in (256, 511, 512, 513, 8191, 20000):
        run_case(px, [1], [n], 4, 2, d, dtype, 4, causal=True, cap=30.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 40])
def test_rows_that_see_nothing(px, d, dtype):
    """More queries than keys under the causal mask, no keys, no queries; zeros come back."""
    for causal in (False, True):
        run_case(px, [70, 3, 0, 5, 200, 1], [30, 0, 9, 5, 1, 0], 4, 2, d, dtype, 5, causal=causal, bias=True)
    q, k, v = inputs([4], [0], 2, 2, d, dtype, 6)
    o = px.varlen_attention_scores(q, k, v, bounds([4]), bounds([0]), 2, 2, d, 0.125, causal=True)
    assert (o == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 24])
def test_prefixes(px, d, dtype):
    """Prefixes of nothing, within a tile, past the queries and past the keys."""
    run_case(px, [300, 129, 64, 70, 90, 1], [300, 200, 64, 70, 90, 500], 4, 2, d, dtype, 7, causal=True, cap=10.0,
             bias=True, prefix=[0, 77, 64, 1000, -5, 3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_segments(px, dtype):
    """More segments than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(8)
    for count in (64, 65, 1100):
        q_len = [int(n) for n in rng.integers(0, 6, count)]
        k_len = [int(n) + int(m) for n, m in zip(q_len, rng.integers(0, 40, count))]
        run_case(px, q_len, k_len, 2, 1, 64, dtype, 9, causal=True, bias=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_strides_and_alignment(px, d, dtype):
    """q, k and v as columns of packed rows, 16-byte aligned and not; o strided too."""
    heads, kv, q_len = 4, 2, [100, 37]
    n = sum(q_len)
    gen = torch.Generator("cuda").manual_seed(10)
    for pad in (0, 8, 3):
        packed = torch.randn((n, (heads + 2 * kv) * d + pad), device="cuda", generator=gen).to(dtype)
        q, k, v = (packed[:, pad + a * d:pad + b * d] for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
        wide = torch.full((n, heads * d + 16 + pad), 9.0, dtype=dtype, device="cuda")
        o = wide[:, pad:pad + heads * d]
        px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(q_len), heads, kv, d, 0.1, cap=8.0, causal=True, out=o)
        want, tol = formula(q, k, v, q_len, q_len, heads, kv, d, 0.1, 8.0, None, True)
        check(o, want, tol, f"pad {pad}")
        assert (wide[:, :pad] == 9.0).all() and (wide[:, pad + heads * d:] == 9.0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 72])
def test_hidden_keys_may_hold_anything(px, d, dtype, bad):
    """Infinite and NaN keys and values that the mask hides change nothing; seen ones
    reach the rows that see them and no other."""
    for q_len, k_len, at in (([200], [200], 190), ([3], [700], 699), ([4], [40], 38), ([300, 60], [300, 60], 130)):
        q, k, v = inputs(q_len, k_len, 4, 2, d, dtype, 11)
        k[at, :d // 2] = bad
        v[at, 3] = bad
        o = px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(k_len), 4, 2, d, 0.1, causal=True, cap=15.0)
        clean_k, clean_v = k.clone(), v.clone()
        clean_k[at], clean_v[at] = 0.0, 0.0
        want, tol = formula(q, clean_k, clean_v, q_len, k_len, 4, 2, d, 0.1, 15.0, None, True)
        # rows of the first segment whose position is below the bad key's
        hidden = at - (k_len[0] - q_len[0])
        check(o[:hidden], want[:hidden], tol[:hidden], "rows before")
        check(o[q_len[0]:], want[q_len[0]:], tol[q_len[0]:], "the next segment")
        assert not torch.isfinite(o[hidden:q_len[0], 3].float()).any(), "a value seen is not hidden"


def test_value_that_only_later_rows_see(px):
    """A NaN value in the last tile, seen by the last row alone, in fp32 and bf16."""
    for dtype in DTYPES:
        q, k, v = inputs([256], [256], 2, 2, 64, dtype, 12)
        v[255] = math.nan
        o = px.varlen_attention_scores(q, k, v, bounds([256]), bounds([256]), 2, 2, 64, 0.125, causal=True)
        assert torch.isfinite(o[:255].float()).all() and torch.isnan(o[255].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_every_size(px, dtype):
    """All scores very small (no seen key may be lost), very large, and equal."""
    for gain, cap in ((0.0, 0.0), (1e-3, 0.0), (30.0, 0.0), (30.0, 50.0), (100.0, 30.0)):
        run_case(px, [130, 1], [130, 900], 4, 2, 64, dtype, 13, causal=True, cap=cap, gain=gain)
    # Falling scores: every later tile lies far below the first, and rising ones.
    q = torch.zeros((2, 64), device="cuda").to(dtype)
    q[:, 0] = 1.0
    k = torch.zeros((600, 64), device="cuda").to(dtype)
    for sign in (1.0, -1.0):
        k[:, 0] = (sign * torch.arange(600, device="cuda")).to(dtype)
        v = torch.randn((600, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(14)).to(dtype)
        o = px.varlen_attention_scores(q, k, v, bounds([2]), bounds([600]), 1, 1, 64, 3.0)
        want, tol = formula(q, k, v, [2], [600], 1, 1, 64, 3.0)
        check(o, want, tol, f"sign {sign}")


def test_same_call_same_bits_and_no_workspace_left_over(px):
    """The same call twice, with a dirtied workspace of a larger call between."""
    q, k, v = inputs([1, 1, 1], [5000, 300, 1], 8, 2, 128, torch.bfloat16, 15)
    ws = px.attention_scores_workspace(3, 3, 5301, 8, 2, 128)
    args = (q, k, v, bounds([1, 1, 1]), bounds([5000, 300, 1]), 8, 2, 128, 0.1)
    a = px.varlen_attention_scores(*args, causal=True, workspace=ws)
    ws.fill_(255)
    b = px.varlen_attention_scores(*args, causal=True, workspace=ws)
    assert torch.equal(a, b)


def test_workspace_never_falls(px):
    size = px.lib.pxs_attention_scores_workspace_bytes
    sizes = [1, 2, 7, 64, 65, 1000, 4096, 70000]
    for heads, kv, d in ((1, 1, 64), (16, 4, 128), (32, 8, 256)):
        for a, b in zip(sizes, sizes[1:]):
            for other in sizes:
                assert size(a, other, other, heads, kv, d) <= size(b, other, other, heads, kv, d)
                assert size(other, a, other, heads, kv, d) <= size(other, b, other, heads, kv, d)
                assert size(other, other, a, heads, kv, d) <= size(other, other, b, heads, kv, d)


@pytest.mark.parametrize("d", [64, 100, 128])
def test_fp32_values_of_every_magnitude(px, d):
    """fp32 operands that three bf16 terms do not hold, in all rows, in some, and beside others:
    values near the least normal number, keys and queries past 2^50, and ordinary ones."""
    heads, kv, q_len, k_len = 4, 2, [150, 1, 40], [150, 600, 300]
    for what in ("tiny values", "some tiny values", "large keys", "one large query", "values from 1e-30 to 1e30"):
        q, k, v = inputs(q_len, k_len, heads, kv, d, torch.float32, 16)
        scale = 1.0 / math.sqrt(d)
        if what == "tiny values":
            v *= 2.0 ** -118
        elif what == "some tiny values":
            v[::7] *= 2.0 ** -118
            v[:, 5] *= 2.0 ** -118
        elif what == "large keys":
            k *= 2.0 ** 55
            scale *= 2.0 ** -55
        elif what == "one large query":
            q[3] *= 2.0 ** 60
        else:
            v *= torch.logspace(-30, 30, d * kv, device="cuda")
        print(f"[scores] fp32 {what} d={d}", flush=True)
        o = px.varlen_attention_scores(q, k, v, bounds(q_len), bounds(k_len), heads, kv, d, scale, causal=True)
        want, tol = formula(q, k, v, q_len, k_len, heads, kv, d, scale, causal=True)
        # (a weight of a few 2^-126 less than the largest is 0: at most that much of the values)
        check(o, want, tol + 2.0 ** -120 * float(v.abs().max()), what)
    assert torch.isfinite(o).all()
