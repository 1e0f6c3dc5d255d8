"""Tree attention (pxs_tree_attention) of more than a million rows, up to what its header names."""

import ctypes as C

import pytest
import torch

import pxs
from test_draft_step_refusals import TREE

BF16 = torch.bfloat16


@pytest.mark.parametrize("change", [
    dict(total_q=2 ** 28, heads=16, kv=16, d=8), dict(total_q=2 ** 24, heads=9, kv=9, d=8), dict(nseg=2 ** 24, heads=4, kv=2)])
def test_grids_too_large_are_refused(change):
    lib = pxs.load_library()
    wide = dict(ld_q=1024, ld_k=1024, ld_v=1024, ld_kc=1024, ld_vc=1024, ld_o=1024, cache_rows=1000)
    assert lib.pxs_tree_attention(*{**TREE, **wide, **change}.values()) == pxs.PXS_ERR_ARG
    assert "grid too large" in lib.pxs_last_error().decode()


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows", [(BF16, 1_100_000), (torch.float32, 1_060_000), (BF16, 4_000_000)])
def test_more_than_a_million_rows(px, dtype, rows):
    """Sequences of 50 tokens over up to 64 cached keys that they share: those at both ends hold what they hold alone."""
    heads, d, each, keys = 16, 8, 50, 200
    segs = rows // each
    assert rows % each == 0 and rows * heads > 2 ** 24 and rows * heads // 8 <= 2 ** 23 and segs * heads <= 2 ** 23
    print(f"[tree limits] {rows} rows {dtype}", flush=True)
    gen = torch.Generator("cuda").manual_seed(61)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dtype)  # noqa: E731
    q, k, v, kc, vc = rand(rows, heads * d), rand(rows, heads * d), rand(rows, heads * d), rand(keys, heads * d), rand(keys, heads * d)
    at = torch.arange(rows, device="cuda") % each
    parents = torch.where(at > 0, (torch.rand(rows, device="cuda", generator=gen) * at).floor().long().clamp_max(at - 1), -1).int()
    cu = torch.arange(0, rows + 1, each, device="cuda")
    start = torch.randint(0, keys - 64, (segs,), device="cuda", generator=gen)
    length = torch.randint(0, 65, (segs,), device="cuda", generator=gen)
    whole = px.tree_attention(q, k, v, cu, parents, kc, vc, start, length, heads, heads, d, 0.3)
    assert bool(torch.isfinite(whole).all())
    for first in (0, segs // 2, segs - 40):
        s, r = slice(first, first + 40), slice(first * each, (first + 40) * each)
        part = px.tree_attention(q[r], k[r], v[r], cu[s.start:s.stop + 1] - r.start, parents[r], kc, vc, start[s], length[s], heads,
                                 heads, d, 0.3)
        assert torch.equal(whole[r], part)
