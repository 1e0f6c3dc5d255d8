"""The RMS norm (pxs_rms_norm, pxs_rms_norm_i8) of more rows than it has workgroups, where each
takes several, and of rows that are stored past the caches (more than 32 MB): every row against
the formula, with test_gpu_rms_norm.py's tolerances."""

import numpy as np
import pytest
import torch

import pxs
from test_gpu_rms_norm import BF16, EPS, F32, LEAST, U, formula, inputs, near, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


@pytest.mark.parametrize("rows,channels,x_dtype,res_dtype", [
    (17000, 300, BF16, F32), (5003, 1370, BF16, BF16), (9001, 1370, F32, None), (5000, 2600, BF16, F32), (4500, 5000, F32, BF16),
    (4300, 8200, BF16, None), (4200, 17000, BF16, F32)])
def test_more_rows_than_workgroups(px, rows, channels, x_dtype, res_dtype):
    print(f"[rms norm rows] {rows} x {channels} {x_dtype} + {res_dtype}", flush=True)
    x, residual, gamma = inputs(rows, channels, x_dtype, res_dtype, rows)
    run(px, x, residual, gamma)


@pytest.mark.parametrize("channels", [1024, 1371, 2600, 8201])
@pytest.mark.parametrize("start", [0, 1])
@pytest.mark.parametrize("y_dtype", [F32, BF16])
def test_rows_past_the_caches(px, y_dtype, start, channels):
    """y of more than 32 MB, from any element; nothing around it is written."""
    rows = (34 << 20) // (channels * (2 if y_dtype is BF16 else 4)) + 1
    assert rows * channels * (2 if y_dtype is BF16 else 4) > 32 << 20
    print(f"[rms norm past] {rows} x {channels} {y_dtype} from {start}", flush=True)
    x, _, gamma = inputs(rows, channels, BF16, None, 31)
    room = torch.full((rows * channels + 4,), 77.0, device="cuda").to(y_dtype)
    px.rms_norm(x, EPS, gamma, out=room[start:start + rows * channels].view(rows, channels))
    got = room[start:start + rows * channels].view(rows, channels)
    for first in range(0, rows, 2048):
        part = slice(first, min(first + 2048, rows))
        _, y, _, _ = formula(x[part], None, gamma, EPS)
        tol = 3 * U * np.abs(y) + LEAST
        if y_dtype is BF16:
            tol = tol + 2.0 ** -8 * (np.abs(y) + tol) + 2.0 ** -134
        near(got[part], y, tol)
    assert (room[:start] == 77.0).all() and (room[start + rows * channels:] == 77.0).all()
