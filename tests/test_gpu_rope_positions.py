"""Rotary positions of token sequences (pxs_rope_positions) against the
formula in 64 bits.

Tolerances.  With u = 2^-24 (half a step of fp32, relative): the angle's rest
is rounded once (at most u / 2 of a quarter turn's half, 0.8 u in radians), sine
and cosine are within 2 u, the magnitude's product u, the two products and the
sum 2 u: an output of a pair (a, b) is off by at most 6 u (|a| + |b|) |magnitude|.
bf16 outputs are rounded once more, by 2^-8 of the value."""

import numpy as np
import pytest
import torch

import pxs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LAYOUTS = {"interleaved": pxs.ROPE_INTERLEAVED, "half": pxs.ROPE_HALF}


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def turned(x, positions, freq, heads, dim, layout, magnitude):
    """-> (values, |a| + |b| of their pairs), float64."""
    r = 2 * len(freq)
    v = x.astype(np.float64).reshape(len(x), heads, dim)
    a_at, b_at = (np.arange(0, r, 2), np.arange(1, r, 2)) if layout == "interleaved" else \
        (np.arange(r // 2), np.arange(r // 2, r))
    # longdouble: the reduction of far angles loses nothing
    angle = (positions.astype(np.longdouble)[:, None] * freq.astype(np.longdouble)[None, :])
    cos, sin = (f(angle).astype(np.float64)[:, None, :] * magnitude for f in (np.cos, np.sin))
    y, size = v.copy(), np.zeros_like(v)
    a, b = v[..., a_at], v[..., b_at]
    y[..., a_at], y[..., b_at] = a * cos - b * sin, a * sin + b * cos
    size[..., a_at] = size[..., b_at] = (np.abs(a) + np.abs(b)) * abs(magnitude)
    return y.reshape(len(x), -1), size.reshape(len(x), -1)


def check(got, want, size, bf16, what):
    off = np.abs(got.double().cpu().numpy() - want)
    tol = 6 * U * size
    if bf16:
        tol = tol + 2.0 ** -8 * (np.abs(want) * (size > 0) + tol)
    assert (off <= tol).all(), f"{what}: {(off - tol).max():.3e} over"


CASES = [  # rows, heads, head_dim, rotary
    (1, 1, 2, 2), (1, 20, 128, 128), (5, 3, 64, 64), (67, 16, 64, 32), (130, 7, 80, 48), (33, 2, 96, 96),
    (9, 5, 40, 6), (3, 1, 1024, 1024), (600, 4, 128, 64), (257, 24, 64, 64), (11, 2, 7, 4),
]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,heads,dim,rotary", CASES)
def test_rope_positions(px, rows, heads, dim, rotary, dtype, layout):
    gen = torch.Generator("cuda").manual_seed(rows + dim)
    for wide, start in ((heads * dim, 0), (heads * dim + 24, 8), (heads * dim + 5, 3)):
        print(f"[rope] {rows} x {heads} x {dim} ({rotary}) {layout} {dtype} at {start} of {wide}", flush=True)
        x = torch.randn((rows, wide), device="cuda", generator=gen).to(dtype)[:, start:start + heads * dim]
        pos = torch.randint(-50, 200000, (rows,), device="cuda", generator=gen).to(torch.int32)
        freq = px.rope_frequencies(rotary, 10000.0, 4.0, 4096.0, 1.0, 32.0)
        out = torch.full((rows + 1, heads * dim), 7.0, dtype=dtype, device="cuda")
        px.rope_positions(x, pos, freq, heads, dim, LAYOUTS[layout], 1.25, out=out[:rows])
        want, size = turned(x.float().cpu().numpy(), pos.cpu().numpy(), freq.cpu().numpy(), heads, dim, layout, 1.25)
        check(out[:rows], want, size, dtype == torch.bfloat16, f"{layout} {dtype}")
        assert (out[rows:] == 7.0).all()
        rest = np.tile(np.arange(dim) >= rotary, heads)
        np.testing.assert_array_equal(out[:rows].float().cpu().numpy()[:, rest], x.float().cpu().numpy()[:, rest])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_on_a_packed_projection(px, dtype, layout):
    """The q and k heads of [rows, q | k | v], in place: the same bits as out of
    place, and v as it was."""
    gen = torch.Generator("cuda").manual_seed(5)
    rows, heads, dim = 300, 20, 64
    qkv = torch.randn((rows, heads * dim + 4 * dim), device="cuda", generator=gen).to(dtype)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32) * 97
    freq = px.rope_frequencies(dim)
    want = px.rope_positions(qkv[:, :heads * dim], pos, freq, heads, dim, LAYOUTS[layout])
    v = qkv[:, heads * dim:].clone()
    px.rope_positions(qkv[:, :heads * dim], pos, freq, heads, dim, LAYOUTS[layout], out=qkv[:, :heads * dim])
    assert torch.equal(qkv[:, :heads * dim], want) and torch.equal(qkv[:, heads * dim:], v)


def test_positions_at_the_ends_of_their_range(px):
    """-2^31 and 2^31 - 1, every angle of the quarter turns, frequencies 0 and above 1."""
    pos = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0, 1, -1, 2, 3, 4, 5, 6, 7, 123456789], dtype=torch.int32, device="cuda")
    freq = torch.tensor([1.0, 0.0, 1.5707963267948966, 0.7853981633974483, 1e-4, 3.0, 6.283185307179586, 0.1],
                        dtype=torch.float64, device="cuda")
    x = torch.randn((12, 16), device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    for layout in LAYOUTS:
        y = px.rope_positions(x, pos, freq, 1, 16, LAYOUTS[layout])
        want, size = turned(x.cpu().numpy(), pos.cpu().numpy(), freq.cpu().numpy(), 1, 16, layout, 1.0)
        # position * frequency is rounded to 53 bits: up to 2^32 radians times 2^-53, twice
        off = np.abs(y.double().cpu().numpy() - want)
        assert (off <= (6 * U + 2.0 ** -19) * size).all()
        near = np.abs(pos.cpu().numpy().astype(np.int64)) < 10
        assert (off[near] <= 6 * U * size[near]).all()


def test_empty_rows(px):
    freq = px.rope_frequencies(64)
    y = px.rope_positions(torch.empty((0, 128), device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), freq, 2, 64)
    assert y.shape == (0, 128)
