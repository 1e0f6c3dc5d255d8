"""Every kernel of the 4-bit linears at one to nine and more stages of K, in every epilogue: the tile that the
host's rule picks for a size is named beside it, so that a new rule cannot leave a kernel without a test.

Tolerances as in test_gpu_linear_mxfp4.py; activations as derived in test_gpu_linear_i8_tiles.py (they go
through the same exponential and reciprocal), inside test_gpu_linear_i8.bounds.  The references' products are
taken in 64 bits on the GPU, with sums of at most 4,096 terms, exact to 2^-52 of the terms' sizes."""

import ctypes as C

import numpy as np
import pytest
import torch

import pxs
from test_gpu_linear_i8 import ACT, U, bounds, check
from test_gpu_linear_mxfp4 import BF16, F32, gpu, random_codes, values

# rows, cin, cout, (tile rows, channels, stages of K)
SIZES = [
    (5, 4240, 33, (16, 16, 0)), (32, 144, 4100, (32, 16, 0)), (40, 400, 2810, (64, 16, 0)), (64, 1400, 2810, (64, 16, 0)),
    # few rows of many channels
    (1, 4096, 14336, (32, 64, 2)), (16, 2000, 16000, (32, 64, 2)), (16, 1025, 20000, (64, 64, 4)),
    (33, 2000, 5001, (32, 64, 2)), (64, 2000, 5000, (32, 64, 2)),
    # four groups take every fourth 256 of K
    (66, 305, 100, (32, 64, 2)), (65, 544, 100, (32, 64, 2)), (65, 774, 100, (32, 64, 2)), (67, 1025, 100, (32, 64, 2)),
    (66, 1281, 100, (32, 64, 2)), (65, 1589, 100, (32, 64, 2)), (67, 1808, 260, (32, 64, 2)), (67, 2116, 101, (32, 64, 2)),
    (87, 8192, 1024, (32, 64, 2)),
    (96, 3, 100, (64, 64, 4)), (72, 277, 100, (64, 64, 4)), (100, 544, 4100, (64, 64, 4)), (1651, 775, 260, (64, 64, 4)),
    (101, 1025, 4100, (64, 64, 4)), (102, 1295, 4100, (64, 64, 4)), (97, 2094, 4100, (64, 64, 4)),
    (1158, 1, 5000, (128, 128, 2)), (710, 273, 4100, (128, 128, 2)), (6589, 760, 260, (128, 128, 2)),
    (6573, 797, 260, (128, 128, 2)), (6555, 1051, 260, (128, 128, 2)), (4739, 1370, 1021, (128, 128, 2)),
    (7248, 2082, 516, (128, 128, 2)), (1370, 1024, 4096, (128, 128, 2)),
    (6574, 1153, 260, (128, 128, 3)), (6738, 1281, 260, (128, 128, 3)), (6581, 1545, 260, (128, 128, 3)),
    (6557, 1856, 260, (128, 128, 3)), (2801, 4000, 1021, (128, 128, 3)),
    (3115, 5, 4100, (256, 256, 2)), (7693, 257, 1540, (256, 256, 2)), (8064, 519, 1540, (256, 256, 2)),
    (3106, 772, 4100, (256, 256, 2)), (7608, 1041, 1540, (256, 256, 2)), (5843, 2062, 2052, (256, 256, 2)),
]
TILES = {(16, 16, 0), (32, 16, 0), (64, 16, 0), (32, 64, 2), (64, 64, 4), (128, 128, 2), (128, 128, 3), (256, 256, 2)}


def tile(lib, rows, cin, cout):
    out = (C.c_int * 3)(-1, -1, -1)
    assert lib.pxs_linear_mxfp4_tile(rows, cin, cout, out) == pxs.PXS_OK
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
        assert tile(lib, max(rows, 1), max(cin, 1), max(cout, 1)) in TILES


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cin,cout,which", SIZES)
def test_tile_in_every_epilogue(px, rows, cin, cout, which):
    print(f"[mxfp4 tile] {rows} x {cin} -> {cout} on {which}", flush=True)
    x, w = random_codes(rows, cin, 61), random_codes(cout, cin, 62)
    rng = np.random.default_rng(63)
    bias = rng.standard_normal(cout).astype(np.float32)
    args = (*map(gpu, x), *map(gpu, w), cin, gpu(bias))
    xv, wv = gpu(values(*x, cin)), gpu(values(*w, cin)).t().contiguous()
    v = (xv @ wv).cpu().numpy() + bias.astype(np.float64)
    size = (xv.abs() @ wv.abs()).cpu().numpy()
    bound = 2 * (cin + 8) * U * size + U * np.abs(v) + 2.0 ** -126
    for act, dtype in (("none", F32), ("none", BF16), ("gelu", BF16), ("silu", F32)):
        y = px.linear_mxfp4(*args, act=ACT[act], dtype=dtype)
        check(y, *bounds(v, bound, act, "bf16" if dtype is BF16 else "f32"), f"{act} {dtype}")
    res = rng.standard_normal((rows, cout)).astype(np.float32)
    residual = gpu(res)
    px.linear_mxfp4_residual(*args, residual)
    want = res + v
    check(residual, want, bound + U * (np.abs(want) + bound), "residual")
    coords = np.zeros((rows, 4), np.int32)
    coords[:, 0] = np.arange(rows) % 2
    block, time = rng.standard_normal(6 * cout).astype(np.float32), rng.standard_normal((2, 6 * cout)).astype(np.float32)
    parts = [np.abs(block)[None, cout:2 * cout] + np.abs(time[coords[:, 0], cout:2 * cout]),
             (block.astype(np.float64) + time)[coords[:, 0], cout:2 * cout]]
    residual = gpu(res)
    px.linear_mxfp4_gate_residual(*args, gpu(coords), gpu(block), gpu(time), cout, residual)
    want = res + v * parts[1]
    check(residual, want, bound * np.abs(parts[1]) + U * (2 * np.abs(v) * parts[0] + np.abs(want)) * 1.01, "gate")
    again = px.linear_mxfp4(*args, dtype=F32)
    assert torch.equal(again, px.linear_mxfp4(*args, dtype=F32))
