"""4-bit linears of up to 2^30 outputs: what a call is run on has a grid that can be launched
(workgroups times threads are counted in 32 bits), and products past the few-rows kernel's grid
(2^27 outputs) against the formula, with test_gpu_linear_mxfp4.py's tolerances."""

import pytest
import torch

import pxs
from test_gpu_linear_i8 import U, bounds, check
from test_gpu_linear_mxfp4 import F32, BF16, gpu, random_codes, reference
from test_gpu_linear_mxfp4_tiles import TILES, tile

THREADS = {which: 256 if which == (64, 64, 4) else 512 for which in TILES}


@pytest.mark.parametrize("cin", [32, 1024, 4096])
@pytest.mark.parametrize("cout", [2 ** 20, 2 ** 26, 2 ** 27 - 16, 2 ** 27 - 1, 2 ** 27, 2 ** 28 + 1, 2 ** 29, 2 ** 30 - 64, 2 ** 30])
def test_every_width_has_a_grid(cout, cin):
    lib = pxs.load_library()
    for rows in (1, 2, 16, 17, 32, 33, 48, 64, 65, 97, 200, 300, 512):
        if rows * cout > 2 ** 38:  # (512 GB of bf16, more than a card holds)
            continue
        which = tile(lib, rows, cin, cout)
        groups = -(-rows // which[0]) * -(-cout // which[1])
        assert groups * THREADS[which] < 2 ** 32, (rows, cin, cout, which)


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cout", [(1, 2 ** 28 + 1), (16, 2 ** 27 + 4), (33, 2 ** 27)])
def test_wide_products(px, rows, cout):
    cin = 32
    print(f"[linear mxfp4 wide] {rows} x {cin} -> {cout}", flush=True)
    x = random_codes(rows, cin, 71)
    gen = torch.Generator("cuda").manual_seed(72)
    codes = torch.randint(0, 256, (cout, 16), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.randint(118, 136, (cout, 16), dtype=torch.uint8, device="cuda", generator=gen)
    bias = torch.randn(cout, device="cuda", generator=gen)
    y = px.linear_mxfp4(*map(gpu, x), codes, scales, cin, bias, dtype=BF16)
    residual = torch.ones((rows, cout), device="cuda")
    px.linear_mxfp4_residual(*map(gpu, x), codes, scales, cin, bias, residual)
    for first in (0, cout // 2 - 50, cout - 150):
        part = slice(first, first + 150)
        v, bound = reference(x, (codes[part].cpu().numpy(), scales[part].cpu().numpy()), bias[part].cpu().numpy(), cin)
        check(y[:, part], *bounds(v, bound, "none", "bf16"), f"store at {first}")
        check(residual[:, part], 1.0 + v, bound + U * (abs(1.0 + v) + bound), f"residual at {first}")
    del codes, scales, bias
    assert bool(torch.isfinite(residual).all()) and residual.dtype is F32
