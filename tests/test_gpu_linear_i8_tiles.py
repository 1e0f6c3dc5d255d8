"""Every kernel of the 8-bit linears, in every epilogue, at ragged sizes: the tile that the host's rule picks
for a size is named beside it, so that a new rule cannot leave a kernel without a test.

Sums in 64 bits are exact (at most 2^31), on the GPU or not.  Tolerances of the sum, scales, bias, residual and
gate as in test_gpu_linear_i8.py.  The activations v r, r = 1 / (1 + 2^e), through the hardware's exponential
and reciprocal (each within 2 u relative, u = 2^-24):
  GELU, e = v (c1 v^2 + c0): off by 4 u |e| (constants, square, sum, product), so 2^e by (2.8 |e| + 2) u; r by
  (1 - r) of that and 3 u (sum and reciprocal); the product adds u: |y| (4 + (1 - r) (2.8 |e| + 2)) u.
  (1 - r) |e| is at most 0.6 for v > 0; for v < 0 |y| |e| <= |v| |e| 2^-|e| <= 0.54 |v|: under 8 u (|v| + 1).
  SiLU, e = -v log2(e), off by 2 u |e|: less.
A slope of at most 1.13 passes an error in v on.  (The bounds of that file, from this form.)"""

import ctypes as C

import numpy as np
import pytest
import torch

import pxs
import workloads as W
from gpu_common import t32, ti32
from test_gpu_linear_i8 import ACT, U, bounds, check, int_rows, ti8

# rows, cin, cout, (tile rows, channels, stages of K)
SIZES = [
    (5, 4240, 33, (16, 16, 0)), (32, 144, 4100, (32, 16, 0)), (40, 400, 2810, (64, 16, 0)),
    (1000, 130, 1021, (128, 128, 1)), (4739, 130, 1021, (192, 128, 1)), (4739, 1370, 516, (128, 128, 1)),
    # four groups take every fourth 128 of K: 3, 5, 6, 7 and 9 of them
    (65, 352, 100, (32, 64, 3)), (130, 528, 1021, (32, 64, 3)), (65, 656, 260, (32, 64, 3)), (300, 784, 100, (32, 64, 3)),
    (257, 1040, 260, (32, 64, 3)),
    (65, 144, 100, (64, 64, 4)), (193, 80, 260, (64, 64, 4)), (700, 272, 1021, (64, 64, 4)),
    (2433, 144, 1540, (128, 64, 3)), (1153, 1296, 1021, (128, 64, 3)), (2370, 2064, 770, (128, 64, 3)),
    (1000, 912, 2052, (128, 128, 2)), (2100, 400, 1021, (128, 128, 2)),
    (2100, 1040, 1021, (128, 128, 3)), (385, 1168, 5000, (128, 128, 3)),
    (1665, 912, 2308, (192, 128, 2)), (5000, 400, 1021, (192, 128, 2)), (1370, 1024, 4096, (192, 128, 2)),
    (1665, 1040, 2308, (192, 128, 3)), (5000, 2064, 772, (192, 128, 3)),
    (3000, 400, 4100, (256, 256, 2)), (8200, 1296, 1021, (256, 256, 2)), (2433, 80, 5000, (256, 256, 2)),
]
TILES = {(16, 16, 0), (32, 16, 0), (64, 16, 0), (128, 128, 1), (192, 128, 1), (32, 64, 3), (64, 64, 4), (128, 64, 3),
         (128, 128, 2), (128, 128, 3), (192, 128, 2), (192, 128, 3), (256, 256, 2)}


def tile(lib, rows, cin, cout, pieces=1):
    out = (C.c_int * 3)(-1, -1, -1)
    assert lib.pxs_linear_i8_tile(rows, cin, cout, pieces, out) == pxs.PXS_OK
    return tuple(out)


def test_sizes_reach_every_tile():
    lib = pxs.load_library()
    for rows, cin, cout, want in SIZES:
        assert tile(lib, rows, cin, cout) == want, (rows, cin, cout)
    assert {want for *_, want in SIZES} == TILES
    # every tile that the rule has for any size is among them
    rng = np.random.default_rng(1)
    for _ in range(4000):
        rows, cin, cout = (int(np.exp(rng.uniform(0, np.log(top)))) for top in (60000, 9000, 9000))
        assert tile(lib, max(rows, 1), max(cin, 1), max(cout, 1), int(rng.integers(0, 2))) in TILES


def test_tile_refusals():
    lib = pxs.load_library()
    out = (C.c_int * 3)()
    for args, text in (((-1, 64, 32), "bad shape"), ((4, 0, 32), "bad shape"), ((4, 64, 0), "bad shape"),
                       ((4, 131072, 32), "131071"), ((4, 64, 2 ** 30 + 1), "2^30 outputs")):
        assert lib.pxs_linear_i8_tile(*args, 1, out) == pxs.PXS_ERR_ARG
        assert text in lib.pxs_last_error().decode()
    assert lib.pxs_linear_i8_tile(4, 64, 32, 1, None) == pxs.PXS_ERR_ARG
    assert tile(lib, 0, 64, 32) == (0, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cin,cout,want", SIZES)
def test_every_tile_in_every_epilogue(rows, cin, cout, want):
    px = pxs.Pxs()
    print(f"[linear_i8] {rows} x {cin} -> {cout} on {want}", flush=True)
    xq, wq = int_rows(86, rows, cin, 1), int_rows(86, cout, cin, 2)
    xs = np.exp(W.normal(86, rows, 3)).astype(np.float32) * np.float32(0.02)
    ws = np.exp(W.normal(86, cout, 4)).astype(np.float32) * np.float32(0.002)
    bias = W.normal(86, cout, 5).astype(np.float32)
    x, w, sx, sw, b = ti8(xq), ti8(wq), t32(xs), t32(ws), t32(bias)
    sums = torch.mm(x.double(), w.double().t().contiguous()).cpu().numpy()
    term = sums * xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None, :]
    v = term + bias.astype(np.float64)[None, :]
    bound = 3.1 * U * np.abs(term) + U * np.abs(v)
    for act, dtype in (("none", torch.float32), ("gelu", torch.bfloat16), ("silu", torch.float32), ("none", torch.bfloat16)):
        y = torch.full((rows + 1, cout), 77.0, dtype=dtype, device="cuda")
        px.linear_i8(x, sx, w, sw, b, ACT[act], out=y[:rows])
        check(y[:rows], *bounds(v, bound, act, "f32" if dtype == torch.float32 else "bf16"), what=f"{act} {dtype}")
        assert (y[rows:] == 77.0).all()
    res = W.normal(86, rows * cout, 6).reshape(rows, cout).astype(np.float32)
    r = t32(np.concatenate([res, res[:1]]))
    px.linear_i8_residual(x, sx, w, sw, b, r[:rows])
    check(r[:rows], res + v, bound + U * np.abs(res + v) + 1e-38, "residual")
    np.testing.assert_array_equal(r[rows:].cpu().numpy(), res[:1])
    coords = np.zeros((rows, 4), np.int32)
    coords[rows // 3:, 0] = 1
    bmod, tmod = W.normal(86, 6 * cout, 7).astype(np.float32), W.normal(86, 2 * 6 * cout, 8).astype(np.float32)
    for offset in (2 * cout, 3):
        r = t32(np.concatenate([res, res[:1]]))
        px.linear_i8_gate_residual(x, sx, w, sw, b, ti32(coords), t32(bmod), t32(tmod), offset, r[:rows])
        gate = bmod.astype(np.float64)[None, offset:offset + cout] + \
            tmod.astype(np.float64).reshape(2, 6 * cout)[coords[:, 0], offset:offset + cout]
        want_r = res + v * gate
        check(r[:rows], want_r, bound * np.abs(gate) + 2.1 * U * np.abs(v * gate) + U * np.abs(want_r) + 1e-38,
              f"gate at {offset}")
        np.testing.assert_array_equal(r[rows:].cpu().numpy(), res[:1])
