"""Attention of drafted trees over a cache (pxs_tree_attention) against the formula in 64
bits, with the tolerances of test_gpu_attention_scores.py (the scores are the same)."""

import math
import random

import numpy as np
import pytest
import torch

import pxs
from test_gpu_attention_scores import B, U, alibi, check

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def parents_of(n, shape, seed):
    host = random.Random(seed)
    if shape == "chain":
        return [t - 1 for t in range(n)]
    if shape == "star":
        return [-1] * n
    if shape == "bad":  # those that are no earlier token count as none
        return [host.choice([t, t + 1, -7, n + 5, 2 ** 31 - 1, -2 ** 31, max(t - 2, -1), t - 1]) for t in range(n)]
    return [-1 if t == 0 else host.randint((t - 1) // 3, t - 1) for t in range(n)]


class Batch:
    """Trees and caches, each sequence's rows somewhere in the cache, NaN between them."""

    def __init__(self, q_len, k_len, heads, kv, d, dtype, seed, shape="tree", cap=0.0, bias=False, gain=2.0, spare=0):
        gen = torch.Generator("cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
        self.q_len, self.k_len, self.heads, self.kv, self.d, self.dtype, self.cap = q_len, k_len, heads, kv, d, dtype, cap
        rows = sum(q_len)
        self.rows = rows
        qkv = torch.full((rows + spare, (heads + 2 * kv) * d), math.nan, device="cuda")
        qkv[:rows] = rand(rows, (heads + 2 * kv) * d)
        qkv[:, :(heads + kv) * d] *= gain
        self.qkv = qkv.to(dtype)
        self.q, self.k, self.v = self.qkv.split([heads * d, kv * d, kv * d], dim=1)
        order = list(range(len(k_len)))
        random.Random(seed).shuffle(order)
        start, at = [0] * len(k_len), 3
        for s in order:
            start[s] = at
            at += k_len[s] + 5
        cache = torch.full((at, 2 * kv * d), math.nan, device="cuda")
        for s in order:
            cache[start[s]:start[s] + k_len[s]] = rand(k_len[s], 2 * kv * d)
        cache[:, :kv * d] *= gain
        self.cache = cache.to(dtype)
        self.kc, self.vc = self.cache.split([kv * d, kv * d], dim=1)
        self.start = start
        self.parents = [parents_of(n, shape, seed + i) for i, n in enumerate(q_len)]
        self.slopes = alibi(heads) if bias else None
        self.depth = []
        for par in self.parents:
            depth = []
            for t, p in enumerate(par):
                depth.append(depth[p] + 1 if 0 <= p < t else 0)
            self.depth.append(depth)
        self.scale = 1.0 / math.sqrt(d)
        dev = dict(device="cuda")
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(q_len)]), dtype=torch.int64, **dev)
        self.t_start, self.t_len = torch.tensor(start, dtype=torch.int64, **dev), torch.tensor(k_len, dtype=torch.int64, **dev)
        self.t_parents = torch.tensor(sum(self.parents, []) + [0] * spare, dtype=torch.int32, **dev)
        self.t_positions = torch.tensor([k_len[i] + x for i, dep in enumerate(self.depth) for x in dep] + [0] * spare,
                                        dtype=torch.int32, **dev)

    def run(self, px, out=None, workspace=None):
        return px.tree_attention(self.q, self.k, self.v, self.cu, self.t_parents, self.kc, self.vc, self.t_start, self.t_len,
                                 self.heads, self.kv, self.d, self.scale, cap=self.cap, slopes=self.slopes,
                                 positions=self.t_positions if self.slopes is not None else None, out=out, workspace=workspace)

    def want(self, k_len=None):
        """-> (values, tolerance) [rows, heads * d]; hidden keys are left out, whatever they hold."""
        heads, kv, d, scale = self.heads, self.kv, self.d, self.scale
        out = torch.zeros((self.rows, heads, d), dtype=torch.float64)
        tol = torch.zeros_like(out)
        qkv, cache = self.qkv.cpu(), self.cache.cpu()
        q_, k_, v_ = qkv.split([heads * d, kv * d, kv * d], dim=1)
        kc, vc = cache.split([kv * d, kv * d], dim=1)
        slopes = None if self.slopes is None else self.slopes.cpu().double()
        q0 = 0
        for i, (n, m) in enumerate(zip(self.q_len, k_len or self.k_len)):
            seen = torch.zeros((n, m + n), dtype=torch.bool)
            seen[:, :m] = True
            for t in range(n):
                c = t
                while c >= 0:
                    seen[t, m + c] = True
                    p = self.parents[i][c]
                    c = p if 0 <= p < c else -1
            where = torch.cat([torch.arange(m), self.k_len[i] + torch.tensor(self.depth[i], dtype=torch.int64)]).double()
            at = slice(self.start[i], self.start[i] + m)
            for h in range(heads):
                col = slice(h // (heads // kv) * d, (h // (heads // kv) + 1) * d)
                q = q_[q0:q0 + n, h * d:(h + 1) * d].double()
                k = torch.cat([kc[at, col], k_[q0:q0 + n, col]]).double()
                v = torch.cat([vc[at, col], v_[q0:q0 + n, col]]).double()
                s = q @ k.T * scale
                e = (q.abs() @ k.abs().T) * scale * (d + 3)
                if self.cap > 0.0:
                    s = self.cap * torch.tanh(s / self.cap)
                    e = e + 8.0 * self.cap
                if slopes is not None:
                    bias = slopes[h] * (where[None, :] - where[m:, None]).abs()
                    s, e = s - bias, e + 4.0 * bias
                e = U * (e + 4.0 * s.abs())
                for row in range(n):
                    see = seen[row]
                    p = torch.exp(s[row, see] - s[row, see].max())
                    total = p.sum()
                    vs, pe = v[see], p * e[row, see]
                    o = p @ vs / total
                    size = p @ vs.abs() / total
                    t = (pe @ vs.abs() + pe.sum() * o.abs()) / total + (int(see.sum()) + 16) * U * size
                    if self.dtype is BF16:
                        t = t + 2 * B * size
                        t = t + B * (o.abs() + t)
                    out[q0 + row, h], tol[q0 + row, h] = o, t + 1e-37
            q0 += n
        return out.flatten(1), tol.flatten(1)


def run_case(px, *args, **kw):
    print(f"[tree] q={args[0][:8]} k={args[1][:8]} segs={len(args[0])} heads={args[2]}/{args[3]} d={args[4]} {args[5]} {kw}", flush=True)
    b = Batch(*args, **kw)
    out = torch.full((b.rows + 2, b.heads * b.d), 55.0, dtype=b.dtype, device="cuda")
    b.run(px, out=out[:b.rows])
    check(out[:b.rows], *b.want(), f"{b.q_len} over {b.k_len}")
    assert (out[b.rows:] == 55.0).all()


MODES = [dict(), dict(cap=20.0), dict(bias=True), dict(cap=5.0, bias=True), dict(cap=2000.0)]
HEADS = [(4, 4, 64), (8, 2, 128), (6, 2, 64), (3, 1, 80), (2, 2, 7), (5, 1, 256), (2, 1, 200), (4, 2, 96), (16, 1, 128)]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,d", HEADS)
def test_trees_over_caches(px, heads, kv, d, dtype, mode):
    """One token to several row tiles, caches of none to some hundred keys."""
    run_case(px, [1, 5, 33, 64, 12], [0, 129, 1, 700, 64], heads, kv, d, dtype, 1, **mode)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,d", HEADS[:5])
def test_few_tokens_over_long_caches(px, heads, kv, d, dtype, mode):
    """Rows that fit a tile; caches cut into chunks, and one of every length around a tile's."""
    run_case(px, [3, 1, 4, 2, 1, 1], [5000, 31, 2000, 128, 0, 65], heads, kv, d, dtype, 2, **mode)


@pytest.mark.parametrize("shape", ["chain", "star", "tree", "bad"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 48])
def test_shapes_of_trees(px, dtype, d, shape):
    run_case(px, [130, 7, 300, 31], [40, 0, 900, 1], 2, 1, d, dtype, 3, shape=shape, bias=shape != "star")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (32, 8)])
def test_one_token(px, dtype, heads, kv):
    """The form for single tokens: over nothing it is the token's own value."""
    for n in (0, 1, 2, 63, 1501):
        run_case(px, [1], [n], heads, kv, 64, dtype, 4 + n)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (F32, 130), (BF16, 64), (BF16, 128), (BF16, 72), (BF16, 33)])
def test_no_cache_at_all(px, dtype, d):
    """Caches of no rows (null pointers), and trees of no tokens between others."""
    b = Batch([3, 0, 70], [0, 0, 0], 4, 2, d, dtype, 11)
    b.kc, b.vc = (torch.empty((0, b.kv * d), dtype=dtype, device="cuda") for _ in range(2))
    check(b.run(px), *b.want(), "no cache")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_sequences(px, dtype):
    """More than a wave holds: the items come from a table."""
    host = random.Random(5)
    for segs in (64, 65, 200):
        run_case(px, [host.randint(0, 5) for _ in range(segs)], [host.choice([0, 3, 40, 130, 700]) for _ in range(segs)], 4, 2, 64,
                 dtype, 6, bias=True)


def test_sequences_past_the_table_kernels_threads(px):
    host = random.Random(7)
    segs = 1100
    run_case(px, [host.randint(0, 2) for _ in range(segs)], [host.choice([0, 3, 40]) for _ in range(segs)], 2, 1, 64, BF16, 8)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_and_small_scores(px, dtype):
    """Scores of hundreds (one key takes all the weight) and of almost nothing."""
    for gain in (20.0, 1e-3):
        run_case(px, [9, 40], [800, 300], 4, 2, 64, dtype, 9, gain=gain)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_hidden_tokens_hold_does_not_matter(px, dtype, d, bad):
    """A token's key and value that are not finite reach it and those below it alone; what the cache holds
    behind a sequence nobody (Batch fills it with NaN)."""
    b = Batch([6, 40, 3], [500, 70, 4000], 4, 2, d, dtype, 10)
    par = [-1, 0, 0, 1, 1, 2]
    b.parents[0] = par
    b.t_parents[:6] = torch.tensor(par, dtype=torch.int32)
    b.v[3], b.k[4], b.v[6 + 39] = bad, math.nan, bad
    got = b.run(px)
    want, tol = b.want()
    poisoned = [3, 4, 6 + 39]
    for row in range(b.rows):
        if row not in poisoned:
            check(got[row], want[row], tol[row], f"row {row}")
    if math.isnan(bad):
        assert torch.isnan(got[3]).all() and torch.isnan(got[4]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(px, dtype):
    """Separate, packed and unaligned rows."""
    heads, kv, d = 4, 2, 64
    b = Batch([20, 3], [300, 1000], heads, kv, d, dtype, 11)
    want, tol = b.want()
    check(b.run(px), want, tol, "packed")
    packed = b.run(px)
    b.q, b.k, b.v, b.kc, b.vc = (t.contiguous() for t in (b.q, b.k, b.v, b.kc, b.vc))
    assert torch.equal(b.run(px), packed)

    def moved(t):  # rows at an odd element
        room = torch.zeros((t.shape[0], t.shape[1] + 3), dtype=dtype, device="cuda")
        room[:, 1:1 + t.shape[1]] = t
        return room[:, 1:1 + t.shape[1]]

    for name in ("q", "k", "v", "kc", "vc"):
        keep = getattr(b, name)
        setattr(b, name, moved(keep))
        check(b.run(px), want, tol, name)
        setattr(b, name, keep)
    out = torch.full((b.rows, heads * d + 3), 9.0, dtype=dtype, device="cuda")
    b.run(px, out=out[:, 1:1 + heads * d])
    check(out[:, 1:1 + heads * d], want, tol, "out")
    assert (out[:, 0] == 9.0).all() and (out[:, 1 + heads * d:] == 9.0).all()


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 64), (BF16, 72)])
def test_padded_batch(px, dtype, d):
    """Rows past the last segment hold anything and keep what they hold; sequences may share a cache."""
    b = Batch([4, 0, 9], [600, 50, 200], 4, 2, d, dtype, 12, spare=7)
    b.start[2] = b.start[0]
    b.t_start[2] = b.t_start[0]
    out = torch.full((b.rows + 7, 4 * d), 3.0, dtype=dtype, device="cuda")
    b.run(px, out=out)
    check(out[:b.rows], *b.want(), "padded")
    assert (out[b.rows:] == 3.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("segs", [3, 70])
def test_bounds_past_the_rows_stay_inside(px, segs, dtype):
    """Bounds that point past the rows, fall or overlap: cut to the rows, or undefined results, but nothing
    around the tensors is touched, and a call that follows is right."""
    rows, keys, d = 48, 3000, 64
    gen = torch.Generator("cuda").manual_seed(13)
    q = torch.randn((rows, d), device="cuda", generator=gen).to(dtype)
    kc, vc = (torch.randn((keys, d), device="cuda", generator=gen).to(dtype) for _ in range(2))
    parents = torch.arange(-1, rows - 1, device="cuda", dtype=torch.int32)
    around = torch.full((rows + 64, d), 3.0, device="cuda").to(dtype)
    o = around[32:32 + rows]

    def call(cu, start, length, out=None):
        fill = segs - (len(cu) - 1)
        cu, start, length = cu + [cu[-1]] * fill, start + [0] * fill, length + [5] * fill
        t = [torch.tensor(x, dtype=torch.int64, device="cuda") for x in (cu, start, length)]
        return px.tree_attention(q, q, q, t[0], parents, kc, vc, t[1], t[2], 1, 1, d, 0.1, out=out)

    good = call([0, rows], [10], [2000])
    far = call([0, rows + 60], [1000], [99999])
    assert torch.equal(far, call([0, rows], [1000], [2000]))
    for cu, start, length in (([0, 40, 8, rows], [0, 100, -5], [3000, -4, 77]), ([0, 20, 48, 10], [2999, 3000, 9999], [5, 5, 5]),
                              ([5, 2, 48, 48], [-2 ** 40, 2 ** 40, 0], [2 ** 40, 7, 2 ** 62]), ([0, -9, 60, 20], [0, 0, 0], [9, 9, 9]),
                              ([0, 48, 0, 48], [0, 0, 0], [3000, 3000, 3000])):
        call(cu, start, length, out=o)
        assert (around[:32] == 3.0).all() and (around[32 + rows:] == 3.0).all()
    assert torch.equal(call([0, rows], [10], [2000]), good)


def test_rows_past_2_31_elements(px):
    """A cache whose element offsets pass 32 bits."""
    kv, d, rows = 8, 128, 1_100_000
    cache = torch.empty((rows, 2 * kv * d), dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(14))
    gen = torch.Generator("cuda").manual_seed(15)
    q = torch.randn((6, 32 * d), device="cuda", generator=gen).bfloat16()
    k, v = (torch.randn((6, kv * d), device="cuda", generator=gen).bfloat16() for _ in range(2))
    cu = torch.tensor([0, 6], device="cuda")
    par = torch.tensor([-1, 0, 0, 1, 2, 2], dtype=torch.int32, device="cuda")
    at, n = rows - 5000, 5000
    one = lambda c, s: px.tree_attention(q, k, v, cu, par, c[:, :kv * d], c[:, kv * d:], torch.tensor([s], device="cuda"),  # noqa: E731
                                         torch.tensor([n], device="cuda"), 32, kv, d, 0.05)
    assert torch.equal(one(cache, at), one(cache[at:].clone(), 0))


@pytest.mark.parametrize("dtype,d", [(F32, 64), (F32, 96), (F32, 160), (F32, 256), (F32, 99), (F32, 201), (BF16, 64), (BF16, 120),
                                     (BF16, 256), (BF16, 99), (BF16, 131)])
def test_long_trees_beside_short_caches(px, dtype, d):
    """Trees of more tokens than a chunk has keys; chunks of unequal shares, rows of several tiles."""
    run_case(px, [400, 1, 140], [1300, 2600, 257], 2, 1, d, dtype, 12, cap=30.0, bias=True)


def test_same_call_same_bits_and_single_tokens_meet_the_scored_attention(px):
    b = Batch([1, 1, 1, 1], [900, 33, 2500, 0], 8, 2, 128, BF16, 16)
    got = b.run(px)
    assert torch.equal(got, b.run(px))
    rows = [torch.cat([b.cache[s:s + n], torch.cat([b.k[i], b.v[i]])[None]]) for i, (s, n) in enumerate(zip(b.start, b.k_len))]
    cat = torch.cat(rows)
    cu_k = torch.tensor(np.concatenate([[0], np.cumsum([n + 1 for n in b.k_len])]), device="cuda")
    other = px.varlen_attention_scores(b.q, cat[:, :256], cat[:, 256:], b.cu, cu_k, 8, 2, 128, b.scale, causal=True)
    want, tol = b.want()
    check(got, want, tol, "tree")
    check(other, want, tol, "scored")


def test_wrong_tensors_are_refused(px):
    b = Batch([4, 2], [10, 20], 2, 1, 64, BF16, 17)
    good = dict(q=b.q, k=b.k, v=b.v, cu_q=b.cu, parents=b.t_parents, k_cache=b.kc, v_cache=b.vc, cache_start=b.t_start,
                cache_len=b.t_len, heads=2, kv_heads=1, head_dim=64, scale=0.1)
    px.tree_attention(**good)
    for change in (dict(q=b.q.cpu()), dict(q=b.q.float()), dict(k=b.k[:3]), dict(v=b.v[:, :32]), dict(v_cache=b.vc[:5]),
                   dict(k_cache=b.kc.t()), dict(cu_q=b.cu.int()), dict(parents=b.t_parents.long()), dict(parents=b.t_parents[:3]),
                   dict(cache_start=b.t_start[:1]), dict(cache_len=b.t_len.int()), dict(slopes=torch.ones(2, device="cuda")),
                   dict(slopes=torch.ones(3, device="cuda"), positions=b.t_positions),
                   dict(slopes=torch.ones(2, device="cuda"), positions=b.t_positions.long()), dict(scale=0.0),
                   dict(out=torch.empty((6, 64), device="cuda", dtype=BF16)),
                   dict(workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(pxs.PxsError):
            px.tree_attention(**{**good, **change})
