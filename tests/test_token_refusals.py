"""Refusals and host functions of the 8-bit linears, the rotary positions and
the scored attention: argument errors are reported before anything reaches a
device, so they are tested without one."""

import ctypes as C
import math

import numpy as np
import pytest

import pxs


@pytest.fixture(scope="module")
def lib():
    return pxs.load_library()


P = C.c_void_p(4096)  # never dereferenced: every call below is refused


def refused(lib, rc, text):
    assert rc == pxs.PXS_ERR_ARG
    assert text in lib.pxs_last_error().decode()


QUANT = dict(dtype=0, x=P, ld=64, rows=4, channels=64, q=P, scales=P, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "bad dtype"), (dict(rows=-1), "bad shape"), (dict(channels=0), "bad shape"),
    (dict(ld=63), "bad shape"), (dict(x=None), "null pointer"), (dict(q=None), "null pointer"),
    (dict(scales=None), "null pointer"), (dict(channels=2 ** 30 + 1, ld=2 ** 31), "2^30 channels")])
def test_quantize_refusals(lib, change, text):
    refused(lib, lib.pxs_quantize_rows_i8(*{**QUANT, **change}.values()), text)


LINEAR = dict(x=P, xs=P, rows=4, cin=64, w=P, ws=P, bias=None, cout=32, act=0, dtype=0, y=P, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=7), "bad dtype"), (dict(act=9), "bad activation"), (dict(rows=-1), "bad shape"),
    (dict(cin=0), "bad shape"), (dict(cout=0), "bad shape"), (dict(cin=131072), "131071"), (dict(x=None), "null pointer"),
    (dict(xs=None), "null pointer"), (dict(w=None), "null pointer"), (dict(ws=None), "null pointer"),
    (dict(y=None), "null pointer"), (dict(rows=2 ** 40, cin=1, cout=2 ** 20), "grid too large"),
    (dict(cin=1, cout=2 ** 31 - 1), "2^30 outputs"), (dict(rows=0, cin=1, cout=2 ** 30 + 1), "2^30 outputs")])
def test_linear_i8_refusals(lib, change, text):
    refused(lib, lib.pxs_linear_i8(*{**LINEAR, **change}.values()), text)


def test_linear_i8_residual_refusals(lib):
    base = dict(x=P, xs=P, rows=4, cin=64, w=P, ws=P, bias=None, cout=32, residual=P, stream=None)
    for change, text in ((dict(residual=None), "null pointer"), (dict(cin=-3), "bad shape"), (dict(cin=200000), "131071")):
        refused(lib, lib.pxs_linear_i8_residual(*{**base, **change}.values()), text)
    gate = dict(x=P, xs=P, rows=4, cin=64, w=P, ws=P, bias=None, cout=32, coords=P, bmod=P, tmod=P, offset=0,
                residual=P, stream=None)
    for change, text in ((dict(offset=-1), "gate offset"), (dict(offset=161), "gate offset"), (dict(coords=None), "null pointer"),
                         (dict(bmod=None), "null pointer"), (dict(tmod=None), "null pointer"), (dict(w=None), "null pointer")):
        refused(lib, lib.pxs_linear_i8_gate_residual(*{**gate, **change}.values()), text)


ROPE = dict(dtype=0, pos=P, freq=P, x=P, ld_x=256, rows=4, heads=4, dim=64, rotary=64, layout=1, mag=1.0, y=P,
            ld_y=256, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "bad dtype"), (dict(layout=2), "bad layout"), (dict(rows=-1), "head_dim"), (dict(heads=0), "heads"),
    (dict(dim=1025, ld_x=9000, ld_y=9000), "1..1024"), (dict(rotary=63), "rotary_dim"), (dict(rotary=66), "rotary_dim"),
    (dict(rotary=0), "rotary_dim"), (dict(ld_x=255), "row stride"), (dict(ld_y=255), "row stride"),
    (dict(mag=math.inf), "magnitude"), (dict(mag=math.nan), "magnitude"), (dict(pos=None), "null pointer"),
    (dict(freq=None), "null pointer"), (dict(x=None), "null pointer"), (dict(y=None), "null pointer"),
    (dict(ld_x=300), "in place")])
def test_rope_positions_refusals(lib, change, text):
    refused(lib, lib.pxs_rope_positions(*{**ROPE, **change}.values()), text)


def test_rope_frequencies(lib):
    def freq(*args):
        out = (C.c_double * (args[0] // 2))()
        assert lib.pxs_rope_frequencies(*args, out) == pxs.PXS_OK
        return np.array(out)

    i = np.arange(32)
    plain = 10000.0 ** (-2.0 * i / 64)
    np.testing.assert_allclose(freq(64, 10000.0, 1.0, 0.0, 0.0, 0.0), plain, rtol=1e-14)
    np.testing.assert_allclose(freq(64, 10000.0, 8.0, 0.0, 0.0, 0.0), plain / 8.0, rtol=1e-14)
    turns = 4096.0 * plain / (2.0 * math.pi)
    keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
    assert keep.min() == 0.0 and keep.max() == 1.0 and ((keep > 0) & (keep < 1)).any()
    np.testing.assert_allclose(freq(64, 10000.0, 8.0, 4096.0, 1.0, 32.0), plain * (keep + (1 - keep) / 8.0), rtol=1e-13)
    np.testing.assert_allclose(freq(64, 10000.0, 1.0, 4096.0, 1.0, 32.0), plain, rtol=1e-14)


@pytest.mark.parametrize("args,text", [
    ((63, 1e4, 1.0, 0.0, 0.0, 0.0), "rotary_dim"), ((0, 1e4, 1.0, 0.0, 0.0, 0.0), "rotary_dim"),
    ((2048, 1e4, 1.0, 0.0, 0.0, 0.0), "rotary_dim"), ((64, 0.0, 1.0, 0.0, 0.0, 0.0), "base"),
    ((64, math.inf, 1.0, 0.0, 0.0, 0.0), "base"), ((64, 1e4, 0.0, 0.0, 0.0, 0.0), "base and factor"),
    ((64, 1e4, 2.0, -1.0, 1.0, 2.0), "original length"), ((64, 1e4, 2.0, 10.0, 2.0, 2.0), "low_turns"),
    ((64, 1e4, 2.0, 10.0, math.nan, 2.0), "low_turns")])
def test_rope_frequencies_refusals(lib, args, text):
    refused(lib, lib.pxs_rope_frequencies(*args, (C.c_double * 1024)()), text)


def test_rope_frequencies_null(lib):
    refused(lib, lib.pxs_rope_frequencies(64, 1e4, 1.0, 0.0, 0.0, 0.0, None), "null pointer")


SCORES = dict(dtype=0, q=P, ld_q=256, k=P, ld_k=128, v=P, ld_v=128, cu_q=P, cu_k=P, nseg=2, total_q=10, total_k=20,
              heads=4, kv=2, d=64, scale=0.125, cap=0.0, slopes=None, causal=1, prefix=None, o=P, ld_o=256, ws=P,
              stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=5), "bad dtype"), (dict(heads=5), "multiple of kv_heads"), (dict(kv=0), "multiple of kv_heads"),
    (dict(heads=131072, kv=1), "65535"), (dict(d=0), "head_dim"), (dict(d=257), "head_dim"), (dict(scale=0.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=math.inf), "cap"), (dict(cap=1e-44), "out of range"),
    (dict(causal=2), "causal"), (dict(causal=0, prefix=P), "prefix"), (dict(nseg=-1), "row counts"),
    (dict(total_q=-1), "row counts"), (dict(total_k=2 ** 31 - 1023), "row counts"),
    (dict(total_q=2 ** 31 - 1024, heads=4, kv=2), "row counts"), (dict(ld_q=255), "row stride"),
    (dict(ld_k=127), "row stride"), (dict(ld_v=127), "row stride"), (dict(ld_o=255), "row stride"),
    (dict(q=None), "null pointer"), (dict(k=None), "null pointer"), (dict(v=None), "null pointer"),
    (dict(o=None), "null pointer"), (dict(cu_q=None), "null pointer"), (dict(cu_k=None), "null pointer"),
    (dict(ws=None), "null pointer"), (dict(ws=C.c_void_p(4104)), "256-byte aligned"),
    (dict(total_q=2 ** 31 - 1024, heads=65535, kv=65535, ld_q=2 ** 23, ld_k=2 ** 23, ld_v=2 ** 23, ld_o=2 ** 23), "grid too large")])
def test_attention_scores_refusals(lib, change, text):
    refused(lib, lib.pxs_varlen_attention_scores(*{**SCORES, **change}.values()), text)


def test_attention_scores_of_nothing(lib):
    for change in (dict(nseg=0), dict(total_q=0)):
        assert lib.pxs_varlen_attention_scores(*{**SCORES, **change}.values()) == pxs.PXS_OK
