"""8-bit linears (pxs_quantize_rows_i8, pxs_linear_i8 and its residual forms)
against the formulas in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32 (relative), 2^-8 half a step of
bf16.  The integer sum is exact, so an output has one rounding to fp32 of the
sum, one for each of the two scales' products and one for the bias:
|error| <= 3.1 u |sum xs ws| + u |value|.  An activation passes an error on by
at most 1.13 times (the GELU's slope; the SiLU's is at most 1.1) and adds its own:
SiLU, v / (1 + e^-v): exp within 2 u relative of itself after a rounding of
v (u |v|, relative to e^-v), a sum, a reciprocal and a product, at most
(|v| + 5) u |silu(v)|, and |v| |silu(v)| <= |v|^2 with e^-v / (1 + e^-v) as a
factor on the part that grows with |v|, under 1: 8 u (|v| + 1) holds.
GELU: the polynomial in tanh's argument is off by 6 u of itself, tanh's
derivative times its argument is at most 0.45, tanhf is within 2 u, and the sum
1 + tanh and two products add 3: under 8 u (|v| + 1) as well.  bf16 outputs are
then rounded once more."""

import numpy as np
import pytest
import torch

import pxs
import workloads as W
from gpu_common import dev, t32, tbf, ti32

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACT = {"none": pxs.ACT_NONE, "gelu": pxs.ACT_GELU_TANH, "silu": pxs.ACT_SILU}


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def quantized(x):
    """The definition in numpy fp32 (each operation rounded once)."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(axis=1)
    bad = ~np.isfinite(x).all(axis=1)
    live = ~bad & (top >= np.float32(2.0 ** -100))
    safe = np.where(live, top, np.float32(1))
    per = np.where(live, np.float32(127) / safe, np.float32(0)).astype(np.float32)
    scale = np.where(live, safe / np.float32(127), np.float32(0)).astype(np.float32)
    scale[bad] = np.nan
    q = np.rint(np.where(live[:, None], x, np.float32(0)) * per[:, None])
    return q.astype(np.int8), scale


def int_rows(seed, rows, cols, stream):
    """Integers over the whole range, -128 among them."""
    v = np.clip(np.rint(W.normal(seed, rows * cols, stream) * 50.0), -128, 127)
    return v.reshape(rows, cols).astype(np.int8)


def activated(v, act):
    if act == "gelu":
        return 0.5 * v * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (v + 0.044715 * v ** 3)))
    return v / (1.0 + np.exp(-v)) if act == "silu" else v


def reference(xq, xs, wq, ws, bias):
    """-> (values before the activation, their error bound) in 64 bits."""
    sums = xq.astype(np.float64) @ wq.astype(np.float64).T
    term = sums * xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None, :]
    v = term + (bias.astype(np.float64)[None, :] if bias is not None else 0.0)
    return v, 3.1 * U * np.abs(term) + U * np.abs(v)


def bounds(v, bound, act, dtype):
    y = activated(v, act)
    tol = bound if act == "none" else 1.13 * bound + 8 * U * (np.abs(v) + 1.0)
    if dtype == "bf16":
        tol = tol + 2.0 ** -8 * (np.abs(y) + tol)
    return y, tol + 1e-38


def check(got, want, tol, what=""):
    off = np.abs(got.detach().double().cpu().numpy() - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol).all(), f"{what}: {off[worst]:.3e} off at {worst}, {tol[worst]:.3e} allowed"


def ti8(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev())


@pytest.mark.parametrize("channels", [1, 7, 8, 64, 512, 515, 520, 1024, 1370, 2048, 4096, 4104, 8192, 9000, 9003])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_rows(px, dtype, channels):
    """Every row width's kernel, whole vectors and not, bit for bit."""
    for rows in (1, 5, 67):
        x = (W.normal(81, rows * channels, 1) * 3.0).reshape(rows, channels).astype(np.float32)
        x[0, channels // 2] = -40.0
        if dtype == "bf16":
            x = W.bf16_round(x)
        q, s = px.quantize_rows((t32 if dtype == "f32" else tbf)(x))
        want_q, want_s = quantized(x)
        np.testing.assert_array_equal(q.cpu().numpy(), want_q)
        np.testing.assert_array_equal(s.cpu().numpy(), want_s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_special_rows(px, dtype):
    """Zeros, tiny and huge rows, ties, infinities and NaN."""
    x = np.zeros((8, 24), np.float32)
    x[1, 3] = 2.0 ** -101          # below what a scale is made of
    x[2, :3] = (2.0 ** -100, 2.0 ** -101, -(2.0 ** -102))
    x[3, 5] = np.inf
    x[4, 6], x[4, 7] = np.nan, 1.0
    x[5, :4] = (3.0e38, -3.0e38, 1.0e38, 1.0)
    x[6] = np.arange(24) - 11.5    # halves: ties of x * (127 / 127)
    x[6, 0] = 127.0
    x[7] = -1.0
    if dtype == "bf16":
        x = W.bf16_round(x)
    q, s = px.quantize_rows((t32 if dtype == "f32" else tbf)(x))
    want_q, want_s = quantized(x)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_strided_and_misaligned_rows(px, dtype):
    """Column slices at every alignment; nothing behind the last row is written."""
    rows, channels = 37, 200
    wide = torch.randn((rows, 3 * channels + 5), device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype)
    for start in (0, 1, 4, 8, 200):
        x = wide[:, start:start + channels]
        q = torch.full((rows + 2, channels), 77, dtype=torch.int8, device="cuda")
        s = torch.full((rows + 2,), 77.0, device="cuda")
        px.quantize_rows(x, out=q[:rows], scales=s[:rows])
        want_q, want_s = quantized(x.float().cpu().numpy())
        np.testing.assert_array_equal(q[:rows].cpu().numpy(), want_q)
        np.testing.assert_array_equal(s[:rows].cpu().numpy(), want_s)
        assert (q[rows:] == 77).all() and (s[rows:] == 77.0).all()


SHAPES = [(1, 1, 1), (1, 16, 8), (3, 15, 5), (2, 17, 33), (5, 127, 64), (16, 128, 16), (17, 144, 100), (64, 1024, 96),
          (65, 1370, 130), (130, 1008, 260), (1, 4096, 1024), (4, 1024, 4096), (33, 2000, 77), (257, 272, 513),
          (700, 1040, 1021), (1370, 256, 1024), (2100, 512, 768), (1370, 1168, 4000), (1000, 1168, 4004)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cin,cout", SHAPES)
def test_linear_i8(px, rows, cin, cout, dtype):
    xq, wq = int_rows(82, rows, cin, 1), int_rows(82, cout, cin, 2)
    xs = np.exp(W.normal(82, rows, 3)).astype(np.float32) * np.float32(0.02)
    ws = np.exp(W.normal(82, cout, 4)).astype(np.float32) * np.float32(0.002)
    bias = W.normal(82, cout, 5).astype(np.float32)
    out = torch.float32 if dtype == "f32" else torch.bfloat16
    for act, b in (("none", None), ("gelu", bias), ("silu", bias)):
        print(f"[linear_i8] {rows} x {cin} -> {cout} {act} {dtype}", flush=True)
        v, bound = reference(xq, xs, wq, ws, b)
        y = torch.full((rows + 1, cout), 77.0, dtype=out, device="cuda")
        px.linear_i8(ti8(xq), t32(xs), ti8(wq), t32(ws), None if b is None else t32(b), ACT[act], out=y[:rows])
        check(y[:rows], *bounds(v, bound, act, dtype), what=f"{rows} x {cin} -> {cout} {act}")
        assert (y[rows:] == 77.0).all()


def test_linear_i8_sum_is_exact_at_the_widest(px):
    """131,071 products of -128 by -128: 2,147,467,264, which 32 bits just hold."""
    cin = 131071
    x = torch.full((2, cin), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, cin), -128, dtype=torch.int8, device="cuda")
    x[1] = 127
    one = torch.ones(3, device="cuda")
    y = px.linear_i8(x, one[:2], w, one, dtype=torch.float32).cpu().numpy()
    np.testing.assert_array_equal(y, np.float32([[16384 * cin] * 3, [-16256 * cin] * 3]))


@pytest.mark.parametrize("rows,cin,cout", [(1, 1024, 1024), (40, 80, 96), (300, 256, 256), (129, 130, 70)])
def test_linear_i8_misaligned_operands(px, rows, cin, cout):
    """Operands, scales, bias and outputs that start off every vector boundary."""
    xq, wq = int_rows(83, rows, cin, 1), int_rows(83, cout, cin, 2)
    xs = np.exp(W.normal(83, rows, 3)).astype(np.float32)
    ws = np.exp(W.normal(83, cout, 4)).astype(np.float32) * np.float32(1e-4)
    bias = W.normal(83, cout, 5).astype(np.float32)

    def shifted(a, by):
        t = torch.from_numpy(np.ascontiguousarray(a))
        buf = torch.zeros(t.numel() + by, dtype=t.dtype, device="cuda")
        buf[by:] = t.reshape(-1).cuda()
        return buf[by:].reshape(t.shape)

    v, bound = reference(xq, xs, wq, ws, bias)
    for by in (1, 4, 8):
        for dtype in (torch.float32, torch.bfloat16):
            y = shifted(np.zeros((rows, cout), np.float32), by).to(dtype) if by != 1 else \
                torch.zeros(rows * cout + 1, dtype=dtype, device="cuda")[1:].reshape(rows, cout)
            px.linear_i8(shifted(xq, by), shifted(xs, by), shifted(wq, by), shifted(ws, by), shifted(bias, by), out=y)
            check(y, *bounds(v, bound, "none", "f32" if dtype == torch.float32 else "bf16"), what=f"shift {by}")


@pytest.mark.parametrize("rows,cin,cout", [(1, 64, 32), (7, 1024, 1024), (250, 1024, 1024), (1237, 272, 320), (90, 33, 18), (1370, 1168, 4000),
                                           (1000, 1168, 4004)])
def test_linear_i8_residual_forms(px, rows, cin, cout):
    xq, wq = int_rows(84, rows, cin, 1), int_rows(84, cout, cin, 2)
    xs = np.exp(W.normal(84, rows, 3)).astype(np.float32) * np.float32(0.02)
    ws = np.exp(W.normal(84, cout, 4)).astype(np.float32) * np.float32(0.002)
    bias = W.normal(84, cout, 5).astype(np.float32)
    res = W.normal(84, rows * cout, 6).reshape(rows, cout).astype(np.float32)
    coords = np.zeros((rows, 4), np.int32)
    coords[rows // 3:, 0] = 1
    bmod, tmod = W.normal(84, 6 * cout, 7).astype(np.float32), W.normal(84, 2 * 6 * cout, 8).astype(np.float32)
    v, bound = reference(xq, xs, wq, ws, bias)
    r = t32(np.concatenate([res, res[:1]]))
    px.linear_i8_residual(ti8(xq), t32(xs), ti8(wq), t32(ws), t32(bias), r[:rows])
    want = res + v
    check(r[:rows], want, bound + U * np.abs(want) + 1e-38, "residual")
    np.testing.assert_array_equal(r[rows:].cpu().numpy(), res[:1])
    for offset in (0, 2 * cout, 5 * cout, 3):
        r = t32(res)
        px.linear_i8_gate_residual(ti8(xq), t32(xs), ti8(wq), t32(ws), t32(bias), ti32(coords), t32(bmod), t32(tmod),
                                   offset, r)
        bm = bmod.astype(np.float64)[None, offset:offset + cout]
        tm = tmod.astype(np.float64).reshape(2, 6 * cout)[coords[:, 0], offset:offset + cout]
        gate = bm + tm
        want = res + v * gate
        # the gate's sum and the product are rounded too
        tol = bound * np.abs(gate) + 2.1 * U * np.abs(v * gate) + U * np.abs(want) + 1e-38
        check(r, want, tol, f"gate at {offset}")


def test_nan_rows_stay_their_own(px):
    """A row with an infinity makes NaN outputs in that row only."""
    x = W.normal(85, 20 * 64, 1).reshape(20, 64).astype(np.float32)
    x[7, 9] = np.inf
    w = W.normal(85, 48 * 64, 2).reshape(48, 64).astype(np.float32)
    q, s = px.quantize_rows(t32(x))
    wq, ws = px.quantize_rows(t32(w))
    y = px.linear_i8(q, s, wq, ws, dtype=torch.float32).cpu().numpy()
    assert np.isnan(y[7]).all() and np.isfinite(np.delete(y, 7, axis=0)).all()


def test_empty_calls(px):
    e = lambda *s, d=torch.float32: torch.empty(s, dtype=d, device="cuda")  # noqa: E731
    q, s = px.quantize_rows(e(0, 64))
    assert q.shape == (0, 64) and s.shape == (0,)
    y = px.linear_i8(q, s, e(32, 64, d=torch.int8), e(32))
    assert y.shape == (0, 32)
