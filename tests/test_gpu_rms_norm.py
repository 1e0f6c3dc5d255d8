"""The RMS norm with the residual's addition (pxs_rms_norm, pxs_rms_norm_i8) against the
formulas: h = residual + x is one rounding in fp32 and one in the residual's type, and the bytes
are those of fp32 arithmetic (test_gpu_linear_i8.quantized of h * gamma), both bit for bit.

Tolerances, u = 2^-24 relative (half a step of fp32): 1 / sqrt(..) comes from 64 bits and is
rounded once, so the scale (max / 127 and its product with that) is off by 3 u, y (two products)
by 3 u, and a bf16 y by 2^-8 (half a step) more; 2^-149 where steps are absolute."""

import numpy as np
import pytest
import torch

import pxs
from test_gpu_linear_i8 import quantized

pytestmark = pytest.mark.gpu
U, LEAST = 2.0 ** -24, 2.0 ** -149
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-6


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def formula(x, residual, gamma, eps):
    """-> (stored h or None, y in 64 bits, q, scales in 64 bits)."""
    h, stored = x.detach().cpu().float(), None
    eps = float(np.float32(eps))  # the call takes a float
    if residual is not None:
        stored = (residual.detach().cpu().float() + h).to(residual.dtype)
        h = stored.float()
    h = h.numpy()
    with np.errstate(all="ignore"):
        inv = 1.0 / np.sqrt((h.astype(np.float64) ** 2).mean(1) + eps)
        g = np.ones(h.shape[1], np.float32) if gamma is None else gamma.cpu().numpy()
        t = (h * g).astype(np.float32)
        q, scale = quantized(t)
        return stored, h.astype(np.float64) * inv[:, None] * g, q, scale.astype(np.float64) * inv


def same_bits(got, want):
    kind = torch.int16 if want.dtype is BF16 else torch.int32
    got, want = got.detach().cpu(), want
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got.view(kind)[~nan], want.view(kind)[~nan])


def near(got, want, tol):
    got = got.detach().double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    off[np.isnan(want) | (got == want)] = 0.0
    assert (off <= tol).all(), f"{off.max():.3e} off"


def run(px, x, residual, gamma, eps=EPS, in_place=False, y_dtype=None):
    stored, y, q, scale = formula(x, residual, gamma, eps)
    for kind in ("i8", "y"):
        res = None if residual is None else residual.clone()
        out = None if residual is None or in_place else torch.empty_like(residual)
        if kind == "i8":
            got_q, got_s = px.rms_norm_i8(x, eps, gamma, res, out)
            np.testing.assert_array_equal(got_q.cpu().numpy(), q)
            near(got_s, scale, 3 * U * np.abs(np.nan_to_num(scale)) + LEAST)
        else:
            got = px.rms_norm(x, eps, gamma, res, out, out_dtype=y_dtype)
            tol = 3 * U * np.abs(np.nan_to_num(y)) + LEAST
            if got.dtype is BF16:
                tol = tol + 2.0 ** -8 * (np.abs(np.nan_to_num(y)) + tol) + 2.0 ** -134
            near(got, y, tol)
        if residual is not None:
            same_bits(res if in_place else out, stored)
            if not in_place:
                same_bits(res, residual.cpu())


def inputs(rows, channels, x_dtype, res_dtype, seed, gamma=True):
    gen = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = (3.0 * rand(rows, channels) * torch.exp(rand(rows, 1))).to(x_dtype)
    residual = None if res_dtype is None else (5.0 * rand(rows, channels)).to(res_dtype)
    return x, residual, torch.exp(0.3 * rand(channels)) * (rand(channels).sign()) if gamma else None


@pytest.mark.parametrize("channels", [1, 7, 8, 9, 64, 500, 512, 513, 1021, 1024, 1370, 2040, 2048, 2049, 4096, 4100, 8192, 8200, 12290, 20001])
@pytest.mark.parametrize("x_dtype,res_dtype", [(F32, None), (BF16, None), (F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
def test_widths(px, x_dtype, res_dtype, channels):
    for rows in (1, 3, 70):
        print(f"[rms norm] {rows} x {channels} {x_dtype} + {res_dtype}", flush=True)
        x, residual, gamma = inputs(rows, channels, x_dtype, res_dtype, channels)
        run(px, x, residual, gamma, in_place=rows == 3)
    run(px, x, residual, None, y_dtype=F32 if x_dtype is BF16 else BF16)


@pytest.mark.parametrize("channels", [24, 1000, 1024, 4096, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(px, dtype, channels):
    """Rows of a wider projection, from any column, and buffers that start anywhere."""
    rows = 37
    gen = torch.Generator("cuda").manual_seed(5)
    for start, pitch in ((0, channels + 24), (8, channels + 16), (1, channels + 3), (3, 2 * channels + 5)):
        wide = torch.randn((rows, pitch), device="cuda", generator=gen).to(dtype)
        flat = torch.randn(rows * channels + 3, device="cuda", generator=gen).to(dtype)
        gamma = torch.rand(channels + 1, device="cuda", generator=gen)
        shift = start % 4
        residual = flat[shift:shift + rows * channels].view(rows, channels)
        x, g = wide[:, start:start + channels], gamma[shift % 2:shift % 2 + channels]
        stored, y, q, scale = formula(x, residual, g, EPS)
        room = torch.full((rows * channels + 5,), 77, dtype=torch.int8, device="cuda")
        out = room[1 + shift:1 + shift + rows * channels].view(rows, channels)
        res_room = torch.full((rows * channels + 5,), 77.0, device="cuda").to(dtype)
        res_out = res_room[1 + shift:1 + shift + rows * channels].view(rows, channels)
        _, scales = px.rms_norm_i8(x, EPS, g, residual, res_out, out=out)
        np.testing.assert_array_equal(out.cpu().numpy(), q)
        near(scales, scale, 3 * U * scale)
        same_bits(res_out, stored)
        for r in (room, res_room):
            assert (r[:1 + shift] == 77).all() and (r[1 + shift + rows * channels:] == 77).all()


@pytest.mark.parametrize("channels", [24, 700, 1024, 4096, 8200, 17000])
def test_special_rows(px, channels):
    """Zeros, rows below and above what fp32 can square, subnormals, ties, infinities and NaN."""
    x = torch.zeros((14, channels))
    x[1, 3] = 2.0 ** -101
    x[2, :3] = torch.tensor([2.0 ** -100, 2.0 ** -101, -(2.0 ** -102)])
    x[3, 5] = float("inf")
    x[4, 6], x[4, 7] = float("nan"), 1.0
    x[5] = 1e30 * torch.linspace(-1, 1, channels)
    x[6] = 3.4e38
    x[7] = 1e-30 * torch.linspace(-1, 1, channels)
    x[8] = 1e-41
    x[9, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5])  # ties of rint
    x[10, 0], x[10, 1] = 3.0e38, -3.0e38
    x[11, 2] = -float("inf")
    x[12, channels - 1] = 1e-20
    x[13] = -0.0
    for eps in (1e-6, 1e-45, 1e5):
        run(px, x.cuda(), None, None, eps)
        run(px, x.cuda(), torch.zeros_like(x).cuda(), torch.full((channels,), 2.0, device="cuda"), eps)
    run(px, x.cuda().bfloat16(), torch.zeros_like(x).cuda().bfloat16(), None)
    # a sum past the residual's largest number is an infinity, and so a NaN row
    run(px, torch.full((2, channels), 3e38, device="cuda"), torch.full((2, channels), 3e38, device="cuda"), None)


def test_i8_rows_are_those_of_the_quantizer(px):
    """With gains of one and no residual: pxs_quantize_rows_i8's bytes."""
    x, _, _ = inputs(100, 1370, BF16, None, 9)
    q, scales = px.rms_norm_i8(x, EPS)
    want, ws = px.quantize_rows(x)
    assert torch.equal(q, want)
    inv = 1.0 / torch.sqrt(x.double().square().mean(1) + EPS)
    near(scales, (ws.double() * inv).cpu().numpy(), 3 * U * (ws.double() * inv).cpu().numpy())


def test_more_than_2_31_values(px):
    """Rows whose offsets pass 32 bits hold what they hold alone."""
    rows, channels = 2_100_001, 1024
    x = torch.empty((rows, channels), dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    residual = torch.empty((rows, channels), dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(4))
    gamma = torch.rand(channels, device="cuda") + 0.5
    last = slice(rows - 50, rows)
    want_res = residual[last].clone()
    want_q, want_s = px.rms_norm_i8(x[last], EPS, gamma, want_res)
    q, s = px.rms_norm_i8(x, EPS, gamma, residual)
    assert torch.equal(q[last], want_q) and torch.equal(s[last], want_s) and torch.equal(residual[last], want_res)


def test_wrong_tensors_are_refused(px):
    x = torch.zeros((4, 64), device="cuda")
    for call in (lambda: px.rms_norm(x.cpu(), EPS), lambda: px.rms_norm(x.double(), EPS), lambda: px.rms_norm(x.t(), EPS),
                 lambda: px.rms_norm(x, EPS, torch.ones(63, device="cuda")), lambda: px.rms_norm(x, EPS, torch.ones(64, device="cuda").bfloat16()),
                 lambda: px.rms_norm(x, EPS, None, x[:3]), lambda: px.rms_norm(x, EPS, None, None, x),
                 lambda: px.rms_norm(x, EPS, None, x.clone(), x.bfloat16()), lambda: px.rms_norm(x, EPS, out=x[:2].clone()),
                 lambda: px.rms_norm(x, EPS, out=x.double()), lambda: px.rms_norm(x, 0.0),
                 lambda: px.rms_norm_i8(x, EPS, out=torch.zeros((4, 64), device="cuda", dtype=torch.uint8)),
                 lambda: px.rms_norm_i8(x, EPS, scales=torch.zeros(3, device="cuda"))):
        with pytest.raises(pxs.PxsError):
            call()
