"""Microscaled 4-bit values and linears (pxs_quantize_mxfp4, pxs_dequantize_mxfp4,
pxs_linear_mxfp4 and its residual forms) against the definitions.

Codes, scales and the values read back are exact, bit for bit.  Products of two values are
exact and their K terms are summed in fp32 in some order: each addition is off by at most
2 u of the sum so far (u = 2^-24, half a step; 2 u where it truncates), which is at most S =
sum |x w|: 2 (K + 8) u S (8: the sums of waves), then u for the bias.  Results below fp32's
least normal number may be zero: 2^-126.  Activations and bf16 outputs as in
test_gpu_linear_i8.bounds."""

import numpy as np
import pytest
import torch

import pxs
from test_gpu_linear_i8 import ACT, U, bounds, check

pytestmark = pytest.mark.gpu
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def blocks_of(x):
    rows, channels = x.shape
    wide = np.zeros((rows, -(-channels // 32) * 32))
    wide[:, :channels] = x
    return wide.reshape(rows, -1, 32)


def quantized(x):
    """-> (codes [rows, 16 blocks], scale bytes [rows, blocks rounded up to 16]) from the definition."""
    w = blocks_of(np.asarray(x, np.float64))
    bad = ~np.isfinite(w).all(axis=2)
    w = np.where(bad[:, :, None], 0.0, w)
    top = np.abs(w).max(axis=2)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    u = np.abs(w) * 2.0 ** -e.astype(np.float64)[:, :, None]
    off = np.abs(u[..., None] - GRID)
    best = off.min(axis=-1, keepdims=True)
    two = off == best                                   # one or two nearest
    even = two & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), two.argmax(-1)).astype(np.uint8)
    code |= (np.signbit(w) & ~bad[:, :, None]).astype(np.uint8) << 3
    code = code.reshape(len(x), -1)
    scales = np.full((len(x), -(-e.shape[1] // 16) * 16), 127, np.uint8)
    scales[:, :e.shape[1]] = np.where(bad, 255, e + 127)
    return code[:, 0::2] | code[:, 1::2] << 4, scales


def values(codes, scales, channels):
    code = np.stack([codes & 15, codes >> 4], axis=2).reshape(len(codes), -1, 32)
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = scales[:, :v.shape[1]].astype(np.float64)
    v = v * np.where(s == 255, np.nan, 2.0 ** (s - 127))[:, :, None]
    return v.reshape(len(codes), -1)[:, :channels]


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def random_rows(rows, channels, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((rows, channels)) * np.exp(spread * rng.standard_normal((rows, 1)))).astype(np.float32)


def check_conversion(px, x):
    """x: an fp32 or bf16 tensor on the GPU."""
    codes, scales = px.quantize_mxfp4(x)
    want_codes, want_scales = quantized(x.detach().float().cpu().numpy())
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(codes.cpu().numpy(), want_codes)
    want = values(want_codes, want_scales, x.shape[1])
    for dtype in (F32, BF16):
        back = px.dequantize_mxfp4(codes, scales, x.shape[1], dtype)
        exact = torch.from_numpy(want).to(F32).to(dtype).double().numpy()
        np.testing.assert_array_equal(back.double().cpu().numpy(), exact)


@pytest.mark.parametrize("channels", [1, 2, 31, 32, 33, 40, 63, 64, 511, 512, 513, 1000, 1024, 1370, 4096])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows(px, dtype, channels):
    for rows in (1, 3, 67):
        check_conversion(px, torch.from_numpy(random_rows(rows, channels, channels)).cuda().to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_border(px, dtype):
    """Each border between two magnitudes and its neighbours on either side, under scales of every size, both
    signs; the block's largest value fixes the scale."""
    half = (GRID[1:] + GRID[:-1]) / 2.0
    at = np.concatenate([half, GRID, [6.5, 7.0, 7.5]]).astype(np.float32)
    step = np.float32(2.0 ** -7 if dtype is BF16 else 2.0 ** -23)
    at = np.concatenate([at, at * (1 + step), at * (1 - step / 2)])
    at = np.concatenate([at, -at])
    rows = []
    for e in (-127, -126, -125, -100, -24, -1, 0, 1, 30, 100, 124, 125):
        for i in range(0, len(at), 31):
            block = np.zeros(32, np.float64)
            part = at[i:i + 31]
            block[:len(part)] = part
            block[31] = 7.0 if np.abs(part).max() > 6.0 else 4.0
            rows.append(block * 2.0 ** e)
    x = np.array(rows)
    x = x[np.abs(x).max(axis=1) < 3.3e38].astype(np.float32)
    check_conversion(px, torch.from_numpy(x).cuda().to(dtype))


def test_special_blocks(px):
    """Zeros, subnormals, one infinity or NaN in a block of a row, the largest numbers, zeros' signs."""
    x = np.zeros((9, 70), np.float32)
    x[1, 3] = np.inf
    x[2, 33], x[2, 40] = np.nan, 1.0
    x[3, 69] = -np.inf
    x[4] = 2.0 ** -149
    x[5, :5] = (2.0 ** -127, 2.0 ** -128, 2.0 ** -129, -(2.0 ** -126), 2.0 ** -149)
    x[6] = 3.4028235e38
    x[7] = -0.0
    x[8, :4] = (1.0, -0.1, 0.1, -0.0)
    check_conversion(px, torch.from_numpy(x).cuda())
    check_conversion(px, torch.from_numpy(x).cuda().bfloat16())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_surroundings(px, dtype):
    """x and y in rows of any stride and start; nothing beside the results is written."""
    for start, channels, pitch in ((0, 96, 104), (8, 64, 80), (1, 65, 67), (5, 300, 311)):
        wide = torch.from_numpy(random_rows(19, pitch, 3)).cuda().to(dtype)
        x = wide[:, start:start + channels]
        codes, scales = px.quantize_mxfp4(x)
        want_codes, want_scales = quantized(x.float().cpu().numpy())
        np.testing.assert_array_equal(codes.cpu().numpy(), want_codes)
        np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
        room = torch.full_like(wide, 77.0)
        px.dequantize_mxfp4(codes, scales, channels, out=room[:, start:start + channels])
        np.testing.assert_array_equal(room[:, start:start + channels].double().cpu().numpy(),
                                      torch.from_numpy(values(want_codes, want_scales, channels)).to(dtype).double().numpy())
        assert (room[:, :start] == 77.0).all() and (room[:, start + channels:] == 77.0).all()


def test_more_than_2_31_values(px):
    rows, channels = 2_200_003, 1000
    x = torch.empty((rows, channels), dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    codes, scales = px.quantize_mxfp4(x)
    want = px.quantize_mxfp4(x[-40:])
    assert torch.equal(codes[-40:], want[0]) and torch.equal(scales[-40:], want[1])
    back = px.dequantize_mxfp4(codes, scales, channels, BF16)
    assert torch.equal(back[-40:], px.dequantize_mxfp4(*want, channels, BF16))


# ---- products ---------------------------------------------------------------------


def random_codes(rows, cin, seed, low=118, high=136):
    """Every code, under scales of a few sizes; bytes past the last block hold anything."""
    rng = np.random.default_rng(seed)
    blocks = -(-cin // 32)
    code = rng.integers(0, 16, (rows, blocks * 32)).astype(np.uint8)
    code[:, cin:] = 0
    scales = rng.integers(0, 256, (rows, -(-blocks // 16) * 16)).astype(np.uint8)
    scales[:, :blocks] = rng.integers(low, high, (rows, blocks))
    if scales.shape[1] > blocks:
        scales[:, blocks] = 255
    return code[:, 0::2] | code[:, 1::2] << 4, scales


def reference(x, w, bias, cin):
    """-> (values before the activation, their error bound) in 64 bits."""
    xv, wv = values(*x, cin), values(*w, cin)
    total = xv @ wv.T
    size = np.abs(xv) @ np.abs(wv).T
    v = total + (bias.astype(np.float64) if bias is not None else 0.0)
    return v, 2 * (cin + 8) * U * size + U * np.abs(v) + 2.0 ** -126


def run_linear(px, rows, cin, cout, act, dtype, bias=True, seed=1):
    print(f"[linear mxfp4] {rows} x {cin} -> {cout} {act} {dtype}", flush=True)
    x, w = random_codes(rows, cin, seed), random_codes(cout, cin, seed + 1)
    b = np.random.default_rng(seed + 2).standard_normal(cout).astype(np.float32) if bias else None
    room = torch.full((rows + 2, cout), 77.0, device="cuda").to(dtype)
    px.linear_mxfp4(*map(gpu, x), *map(gpu, w), cin, gpu(b) if bias else None, ACT[act], out=room[1:1 + rows])
    v, bound = reference(x, w, b, cin)
    y, tol = bounds(v, bound, act, "bf16" if dtype is BF16 else "f32")
    check(room[1:1 + rows], y, tol, f"{rows} x {cin} -> {cout}")
    assert (room[0] == 77.0).all() and (room[-1] == 77.0).all()


@pytest.mark.parametrize("rows,cin,cout", [
    (1, 1, 1), (1, 32, 16), (1, 33, 17), (1, 64, 3), (2, 31, 100), (16, 256, 64), (17, 257, 33), (5, 1024, 4096), (33, 1370, 100),
    (64, 500, 1021), (65, 288, 260), (130, 512, 1021), (300, 1024, 129), (257, 96, 516), (1000, 1370, 1021), (700, 4096, 260),
    (2433, 700, 1540)])
@pytest.mark.parametrize("act,dtype", [("none", F32), ("gelu", BF16), ("silu", F32), ("none", BF16)])
def test_linear(px, rows, cin, cout, act, dtype):
    run_linear(px, rows, cin, cout, act, dtype, bias=act != "none" or dtype is F32)


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_scales_of_every_size(px, rows):
    """Scales from 2^-127 to 2^127 whose products stay ordinary: the bytes' sum is what counts."""
    cin, cout = 300, 70
    x, w = random_codes(rows, cin, 11, 0, 8), random_codes(cout, cin, 12, 244, 255)
    v, bound = reference(x, w, None, cin)
    check(px.linear_mxfp4(*map(gpu, x), *map(gpu, w), cin, dtype=F32), v, bound, "small by large")
    v, bound = reference(w, x, None, cin)
    check(px.linear_mxfp4(*map(gpu, w), *map(gpu, x), cin, dtype=F32), v, bound, "large by small")


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_nan_scales(px, rows):
    """A block without a scale makes its row's, or its channel's, outputs NaN, and no others."""
    cin, cout = 700, 100
    x, w = random_codes(rows, cin, 21), random_codes(cout, cin, 22)
    x[1][1, 3], x[1][rows - 1, 21], w[1][7, 0], w[1][99, 20] = 255, 255, 255, 255
    x[0][1, 48:64] = 0  # zeros without a scale as well
    got = px.linear_mxfp4(*map(gpu, x), *map(gpu, w), cin, dtype=F32).cpu().numpy()
    nan = np.zeros((rows, cout), bool)
    nan[[1, rows - 1]] = True
    nan[:, [7, 99]] = True
    np.testing.assert_array_equal(np.isnan(got), nan)
    v, bound = reference(x, w, None, cin)
    assert (np.abs(got - v)[~nan] <= bound[~nan]).all()


@pytest.mark.parametrize("rows,cin,cout", [(1, 1370, 100), (20, 64, 33), (70, 512, 1021), (400, 1000, 260), (2000, 320, 516)])
def test_residual_and_gate(px, rows, cin, cout):
    """residual += linear, and += gate * linear: one more rounding of the product with the gate (the gate
    itself is a sum of two, rounded) and one of the sum."""
    x, w = random_codes(rows, cin, 31), random_codes(cout, cin, 32)
    rng = np.random.default_rng(33)
    b, res = rng.standard_normal(cout).astype(np.float32), rng.standard_normal((rows, cout)).astype(np.float32)
    v, bound = reference(x, w, b, cin)
    residual = gpu(res)
    px.linear_mxfp4_residual(*map(gpu, x), *map(gpu, w), cin, gpu(b), residual)
    want = res + v
    check(residual, want, bound + U * (np.abs(want) + bound), "residual")
    coords = np.zeros((rows, 4), np.int32)
    coords[:, 0] = rng.integers(0, 2, rows)
    block, time = rng.standard_normal(6 * cout).astype(np.float32), rng.standard_normal((2, 6 * cout)).astype(np.float32)
    for offset in (0, 2 * cout):
        gate = (block.astype(np.float64) + time)[coords[:, 0], offset:offset + cout]
        residual = gpu(res)
        px.linear_mxfp4_gate_residual(*map(gpu, x), *map(gpu, w), cin, gpu(b), gpu(coords), gpu(block), gpu(time), offset, residual)
        want = res + v * gate
        size = np.abs(block)[None, offset:offset + cout] + np.abs(time[coords[:, 0], offset:offset + cout])
        tol = bound * np.abs(gate) + U * (2 * np.abs(v) * size + np.abs(want)) * 1.01
        check(residual, want, tol, f"gate at {offset}")


@pytest.mark.parametrize("rows", [5, 100, 700])
def test_unaligned_outputs(px, rows):
    """y, bias and residual that start anywhere."""
    cin, cout = 256, 68
    x, w = random_codes(rows, cin, 41), random_codes(cout, cin, 42)
    b = np.random.default_rng(43).standard_normal(cout + 1).astype(np.float32)
    for dtype in (F32, BF16):
        room = torch.full((rows * cout + 2,), 77.0, device="cuda").to(dtype)
        px.linear_mxfp4(*map(gpu, x), *map(gpu, w), cin, gpu(b)[1:], out=room[1:-1].view(rows, cout))
        v, bound = reference(x, w, b[1:], cin)
        check(room[1:-1].view(rows, cout), *bounds(v, bound, "none", "bf16" if dtype is BF16 else "f32"))
        assert room[0] == 77.0 and room[-1] == 77.0
    room = torch.zeros(rows * cout + 2, device="cuda")
    px.linear_mxfp4_residual(*map(gpu, x), *map(gpu, w), cin, gpu(b)[1:], room[1:-1].view(rows, cout))
    check(room[1:-1].view(rows, cout), v, bound + U * np.abs(v), "residual")
    assert room[0] == 0.0 and room[-1] == 0.0


def test_outputs_past_2_31(px):
    """A product whose offsets pass 32 bits: rows hold what they hold alone."""
    rows, cin, cout = 540_001, 64, 4004
    codes = torch.randint(0, 256, (rows, 32), dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    scales = torch.full((rows, 16), 127, dtype=torch.uint8, device="cuda")
    w = random_codes(cout, cin, 52)
    y = px.linear_mxfp4(codes, scales, *map(gpu, w), cin)
    v, bound = reference((codes[-33:].cpu().numpy(), scales[-33:].cpu().numpy()), w, None, cin)
    check(y[-33:], *bounds(v, bound, "none", "bf16"))


def test_wrong_tensors_are_refused(px):
    x = torch.zeros((4, 64), device="cuda")
    q, s = px.quantize_mxfp4(x)
    w, ws = px.quantize_mxfp4(torch.ones((32, 64), device="cuda"))
    for call in (lambda: px.quantize_mxfp4(x.cpu()), lambda: px.quantize_mxfp4(x.half()), lambda: px.quantize_mxfp4(x.t()[:, :4]),
                 lambda: px.quantize_mxfp4(x, out=q[:2]), lambda: px.quantize_mxfp4(x, scales=s[:, :8]),
                 lambda: px.dequantize_mxfp4(q, s, 65), lambda: px.dequantize_mxfp4(q, s, 64, out=x[:3]),
                 lambda: px.dequantize_mxfp4(q, s, 64, torch.float16), lambda: px.linear_mxfp4(q, s, w, ws, 65),
                 lambda: px.linear_mxfp4(q, s, w, ws[:3], 64), lambda: px.linear_mxfp4(q, s.int(), w, ws, 64),
                 lambda: px.linear_mxfp4(q, s, w, ws, 64, torch.ones(31, device="cuda")),
                 lambda: px.linear_mxfp4(q, s, w, ws, 64, out=torch.zeros((4, 31), device="cuda")),
                 lambda: px.linear_mxfp4_residual(q, s, w, ws, 64, None, torch.zeros((4, 32), device="cuda").bfloat16())):
        with pytest.raises(pxs.PxsError):
            call()
