"""The tree attention's walks of many key tiles and its joins of many rows (pxs_tree_attention)
against the formula, with the tolerances of test_gpu_attention_tree.py.  Which steps and which
join a case runs on is asked of the host's plan, so that a new rule cannot leave them without a test."""

import ctypes as C
import math
import random

import pytest
import torch

import pxs
from test_gpu_attention_scores import B, U, check
from test_gpu_attention_tree import MODES, Batch

F32, BF16 = torch.float32, torch.bfloat16
LONG_WALK = 6  # steps without a maximum: the first, the last, and the loop's at least twice


def plan(dtype, q_len, k_len, heads, kv, d, cache_rows=None):
    """-> dict(rows, keys, chunk, even, odd, join) of a call on these lengths."""
    out, n = (C.c_int * 6)(), len(q_len)
    rows = sum(k_len) + 5 * n + 3 if cache_rows is None else cache_rows  # Batch's cache
    rc = pxs.load_library().pxs_tree_attention_plan(pxs._DTYPE_CODES[dtype], (C.c_int64 * n)(*q_len), (C.c_int64 * n)(*k_len), n,
                                                    rows, heads, kv, d, out)
    assert rc == pxs.PXS_OK
    return dict(zip(("rows", "keys", "chunk", "even", "odd", "join"), out))


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def want(b):
    """Batch.want() in 64 bits on the GPU, all rows of a head at once, for trees whose values are finite."""
    heads, kv, d = b.heads, b.kv, b.d
    out = torch.zeros((b.rows, heads, d), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    q0 = 0
    for i, (n, m) in enumerate(zip(b.q_len, b.k_len)):
        seen = torch.zeros((n, m + n), dtype=torch.bool)
        seen[:, :m] = True
        for t in range(n):
            c = t
            while c >= 0:
                seen[t, m + c] = True
                p = b.parents[i][c]
                c = p if 0 <= p < c else -1
        seen = seen.cuda()
        where = torch.cat([torch.arange(m), b.k_len[i] + torch.tensor(b.depth[i], dtype=torch.int64)]).double().cuda()
        at, rows = slice(b.start[i], b.start[i] + m), slice(q0, q0 + n)
        for h in range(heads if n else 0):
            col = slice(h // (heads // kv) * d, (h // (heads // kv) + 1) * d)
            q = b.q[rows, h * d:(h + 1) * d].double()
            k = torch.cat([b.kc[at, col], b.k[rows, col]]).double()
            v = torch.cat([b.vc[at, col], b.v[rows, col]]).double()
            s = q @ k.t().contiguous() * b.scale
            e = q.abs() @ k.abs().t().contiguous() * (b.scale * (d + 3))
            if b.cap > 0.0:
                s, e = b.cap * torch.tanh(s / b.cap), e + 8.0 * b.cap
            if b.slopes is not None:
                bias = b.slopes[h].double() * (where[None, :] - where[m:, None]).abs()
                s, e = s - bias, e + 4.0 * bias
            e = U * (e + 4.0 * s.abs())
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(1, keepdim=True))
            p = p / p.sum(1, keepdim=True)
            o, size, pe = p @ v, p @ v.abs(), p * e
            t = pe @ v.abs() + pe.sum(1, keepdim=True) * o.abs() + (seen.sum(1, keepdim=True) + 16) * U * size
            if b.dtype is BF16:
                t = t + 2 * B * size
                t = t + B * (o.abs() + t)
            out[rows, h], tol[rows, h] = o, t + 1e-37
        q0 += n
    return out.flatten(1).cpu(), tol.flatten(1).cpu()


def run_case(px, *args, change=None, **kw):
    print(f"[tree paths] q={args[0][:8]} k={args[1][:8]} segs={len(args[0])} heads={args[2]}/{args[3]} d={args[4]} {args[5]} {kw}",
          flush=True)
    b = Batch(*args, **kw)
    if change is not None:
        change(b)
    out = torch.full((b.rows + 2, b.heads * b.d), 55.0, dtype=b.dtype, device="cuda")
    b.run(px, out=out[:b.rows])
    check(out[:b.rows], *want(b), f"{b.q_len[:8]} over {b.k_len[:8]}")
    assert (out[b.rows:] == 55.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_reference(dtype):
    """The two references agree."""
    for kw in MODES:
        b = Batch([5, 0, 33], [129, 7, 0], 4, 2, 24, dtype, 20, **kw)
        for got, other in zip(want(b), b.want()):
            assert torch.allclose(got, other, rtol=1e-9, atol=1e-12)


# ---- steps without a maximum ---------------------------------------------------------
# trees, caches, heads, key/value heads: one tile with three idle waves; two tiles, the second with three idle
# waves; four waves of rows; a cache that ends inside a tile and one that does not.
WALKS = [([3], [40000], 8, 8), ([3], [39457], 8, 8), ([70, 2], [26000, 9001], 16, 8), ([64, 1], [30016, 4000], 16, 8)]
SIZES = [64, 128, 40, 96, 120]


@pytest.mark.parametrize("d", SIZES)
def test_walks_are_long(d):
    """Even and odd numbers of steps, for every head size."""
    plans = [plan(BF16, *walk, d) for walk in WALKS]
    assert min(p["odd"] for p in plans) >= LONG_WALK and sum(p["even"] >= LONG_WALK for p in plans) >= 2, plans


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("d", SIZES)
@pytest.mark.parametrize("q_len,k_len,heads,kv", WALKS)
def test_long_walks(px, q_len, k_len, heads, kv, d, mode):
    run_case(px, q_len, k_len, heads, kv, d, BF16, 21, **mode)


def waves(batch, rise, period, seed):
    """Scores that climb by `rise` over every `period` keys from the later to the earlier, as the walk goes, and
    fall back: q and k of a head share one direction, with what Batch drew beside it."""
    heads, kv, d = batch.heads, batch.kv, batch.d
    gen = torch.Generator("cuda").manual_seed(seed)
    u = torch.randn(kv, d, device="cuda", generator=gen)
    u /= u.norm(dim=1, keepdim=True)
    size = math.sqrt(rise / batch.scale)
    q = batch.q.float().view(-1, kv, heads // kv, d) * 0.1 + size * u[None, :, None]
    batch.q.copy_(q.flatten(1).to(batch.dtype))
    at = torch.arange(batch.cache.shape[0], device="cuda")
    climb = 1.0 - (at % period).float() / period
    k = batch.kc.float().view(-1, kv, d) * 0.1 + size * climb[:, None, None] * u[None]
    batch.kc.copy_(k.flatten(1).to(batch.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [dict(), dict(cap=2000.0), dict(bias=True)])
@pytest.mark.parametrize("d", [64, 128, 40, 96])
@pytest.mark.parametrize("q_len,k_len,heads,kv", WALKS[1:3])
def test_scores_that_rise_along_the_walk(px, q_len, k_len, heads, kv, d, mode):
    """By e^100 over 1,000 keys: weights past 2^40 of the base, taken again with a maximum, several times a walk."""
    p = plan(BF16, q_len, k_len, heads, kv, d)
    assert (p["odd"] - 1) * p["keys"] / 1000 * 100 > 40 * math.log(2)
    run_case(px, q_len, k_len, heads, kv, d, BF16, 22, change=lambda b: waves(b, 100.0, 1000, 23), **mode)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e30, 1e33, 1e36])
@pytest.mark.parametrize("d", [64, 128, 40, 96])
@pytest.mark.parametrize("q_len,k_len,heads,kv", WALKS[1:3])
def test_large_values_under_rising_scores(px, q_len, k_len, heads, kv, d, size):
    """Unnormalised outputs past 2^118, which are walked again: e^16 and more within a walk, times values of
    2^100 and more."""
    p = plan(BF16, q_len, k_len, heads, kv, d)
    rise = 40.0
    assert math.log2(size) + min((p["odd"] - 1) * p["keys"] / 1000, 1.0) * rise / math.log(2) > 118

    def change(b):
        waves(b, rise, 1000, 25)
        b.vc.copy_((b.vc.float() * size).to(BF16))
        b.v.copy_((b.v.float() * size).to(BF16))

    run_case(px, q_len, k_len, heads, kv, d, BF16, 24, change=change)


# ---- joins of many rows -----------------------------------------------------------------

host = random.Random(26)
JOINS = [([100, 250, 10], [700, 3000, 64]), ([host.randint(3, 9) for _ in range(70)], [host.choice([0, 40, 700, 901]) for _ in range(70)])]
JOIN_HEADS = [(12, 4), (20, 5), (8, 8)]


def test_joins_are_of_rows_each():
    for q_len, k_len in JOINS:
        for heads, kv in JOIN_HEADS:
            q = widened(q_len, heads)
            for dtype in (F32, BF16):
                for d in (64, 99, 256):
                    assert plan(dtype, q, k_len, heads, kv, d)["join"] == 2, (q_len, heads, d)
    assert plan(BF16, [1], [9000], 16, 8, 64)["join"] == 1 and plan(BF16, [400], [50], 16, 8, 64)["join"] == 0


def widened(q_len, heads):
    """As many tokens more in the first tree as the rows take to be many."""
    return [q_len[0] + max(0, -(-4200 // heads) - sum(q_len))] + q_len[1:]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 99, 256, 48])
@pytest.mark.parametrize("heads,kv", JOIN_HEADS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", [0, 1])
def test_many_rows_over_chunked_caches(px, which, dtype, heads, kv, d):
    q_len, k_len = JOINS[which]
    run_case(px, widened(q_len, heads), k_len, heads, kv, d, dtype, 27, cap=30.0 if d == 64 else 0.0)


# ---- the plan's refusals --------------------------------------------------------------------


def test_plan_refusals():
    lib = pxs.load_library()
    lens, out = (C.c_int64 * 2)(3, 1), (C.c_int * 6)()
    good = dict(dtype=1, q=lens, k=lens, nseg=2, cache_rows=10, heads=4, kv=2, d=64, plan=out)
    assert lib.pxs_tree_attention_plan(*good.values()) == pxs.PXS_OK
    for change, text in ((dict(dtype=2), "bad dtype"), (dict(heads=3), "bad heads"), (dict(kv=0), "bad heads"), (dict(d=257), "bad heads"),
                         (dict(nseg=0), "null pointer"), (dict(q=None), "null pointer"), (dict(k=None), "null pointer"),
                         (dict(plan=None), "null pointer"), (dict(cache_rows=-1), "bad cache"), (dict(cache_rows=2), "bad length"),
                         (dict(q=(C.c_int64 * 2)(3, -1)), "bad length"), (dict(q=(C.c_int64 * 2)(2 ** 30, 2 ** 30)), "bad length")):
        assert lib.pxs_tree_attention_plan(*{**good, **change}.values()) == pxs.PXS_ERR_ARG
        assert text in lib.pxs_last_error().decode()
