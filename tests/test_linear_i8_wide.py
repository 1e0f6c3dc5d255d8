"""8-bit linears of up to 2^29 outputs: what a call is run on has a grid that can be launched
(workgroups times threads are counted in 32 bits)."""

import pytest
import torch

import pxs
from test_gpu_linear_i8 import bounds, check, reference
from test_gpu_linear_i8_tiles import TILES, tile

THREADS = {which: 1024 if which[0] == 256 else 256 if which == (64, 64, 4) else 512 for which in TILES}


@pytest.mark.parametrize("pieces", [0, 1])
@pytest.mark.parametrize("cin", [32, 1024, 4096])
@pytest.mark.parametrize("cout", [2 ** 20, 2 ** 26, 2 ** 27 - 16, 2 ** 27 - 1, 2 ** 27, 2 ** 28 + 1, 2 ** 29 - 64, 2 ** 29])
def test_every_width_has_a_grid(cout, cin, pieces):
    lib = pxs.load_library()
    for rows in (1, 2, 16, 17, 32, 33, 48, 64, 65, 97, 128, 200, 300, 512, 1000):
        if -(-rows // 128) * -(-cout // 128) >= 2 ** 23:  # (the header's limit)
            continue
        which = tile(lib, rows, cin, cout, pieces)
        groups = -(-rows // which[0]) * -(-cout // which[1])
        assert groups * THREADS[which] < 2 ** 32, (rows, cin, cout, pieces, which)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cin", [(1, 32), (20, 17)])
def test_wide_products(rows, cin):
    """More outputs than the few-rows kernel's grid holds, in whole pieces and not."""
    px, cout = pxs.Pxs(), 2 ** 28 + 3
    print(f"[linear i8 wide] {rows} x {cin} -> {cout}", flush=True)
    gen = torch.Generator("cuda").manual_seed(81)
    x = torch.randint(-127, 128, (rows, cin), dtype=torch.int8, device="cuda", generator=gen)
    w = torch.randint(-127, 128, (cout, cin), dtype=torch.int8, device="cuda", generator=gen)
    xs, ws = torch.rand(rows, device="cuda", generator=gen), torch.rand(cout, device="cuda", generator=gen)
    y = px.linear_i8(x, xs, w, ws, None, out=torch.full((rows, cout), 77.0, dtype=torch.bfloat16, device="cuda"))
    for first in (0, cout // 2, cout - 100):
        part = slice(first, first + 100)
        v, bound = reference(*(t.cpu().numpy() for t in (x, xs, w[part], ws[part])), None)
        check(y[:, part], *bounds(v, bound, "none", "bf16"), f"at {first}")
