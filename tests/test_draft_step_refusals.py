"""Refusals and host functions of the RMS norm, the 4-bit linears and the tree attention:
argument errors are reported before anything reaches a device, so they are tested without one."""

import ctypes as C
import math

import pytest

import pxs


@pytest.fixture(scope="module")
def lib():
    return pxs.load_library()


P = C.c_void_p(4096)  # never dereferenced: every call below is refused
ODD = C.c_void_p(4104)


def refused(lib, rc, text):
    assert rc == pxs.PXS_ERR_ARG
    assert text in lib.pxs_last_error().decode()


NORM = dict(x_dtype=0, x=P, ld=64, res_dtype=1, residual=P, out=P, rows=4, channels=64, eps=1e-6, gamma=None)
Y = dict(y_dtype=0, y=P, stream=None)
Q = dict(q=P, scales=P, stream=None)
NORM_CHANGES = [
    (dict(x_dtype=2), "bad dtype"), (dict(res_dtype=2), "bad residual dtype"), (dict(rows=-1), "bad shape"),
    (dict(channels=0), "bad shape"), (dict(ld=63), "bad shape"), (dict(channels=2 ** 30 + 1, ld=2 ** 31), "2^30 channels"),
    (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"),
    (dict(residual=None), "both be given"), (dict(out=None), "both be given"), (dict(x=None), "null pointer")]


@pytest.mark.parametrize("change,text", NORM_CHANGES + [(dict(y_dtype=2), "bad dtype"), (dict(y=None), "null pointer")])
def test_rms_norm_refusals(lib, change, text):
    refused(lib, lib.pxs_rms_norm(*{**NORM, **Y, **change}.values()), text)


@pytest.mark.parametrize("change,text", NORM_CHANGES + [(dict(q=None), "null pointer"), (dict(scales=None), "null pointer")])
def test_rms_norm_i8_refusals(lib, change, text):
    refused(lib, lib.pxs_rms_norm_i8(*{**NORM, **Q, **change}.values()), text)


def test_norms_of_nothing(lib):
    none = dict(x=None, residual=None, out=None, rows=0)
    assert lib.pxs_rms_norm(*{**NORM, **Y, **none, "y": None}.values()) == pxs.PXS_OK
    assert lib.pxs_rms_norm_i8(*{**NORM, **Q, **none, "q": None, "scales": None}.values()) == pxs.PXS_OK


def test_mxfp4_row_bytes(lib):
    for channels, codes, scales in ((-1, 0, 0), (0, 0, 0), (1, 16, 16), (32, 16, 16), (33, 32, 16), (512, 256, 16),
                                    (513, 272, 32), (1370, 688, 48), (4096, 2048, 128), (2 ** 31 - 1, 2 ** 30, 2 ** 26)):
        assert lib.pxs_mxfp4_code_bytes(channels) == codes
        assert lib.pxs_mxfp4_scale_bytes(channels) == scales
        if channels > 0:
            assert pxs._mxfp4_bytes(channels) == (codes, scales)


QUANT = dict(dtype=0, x=P, ld=64, rows=4, channels=64, codes=P, scales=P, stream=None)
QUANT_CHANGES = [
    (dict(dtype=2), "bad dtype"), (dict(rows=-1), "bad shape"), (dict(channels=0), "bad shape"), (dict(ld=63), "bad shape"),
    (dict(channels=2 ** 30 + 1, ld=2 ** 31), "2^30 channels"), (dict(x=None), "null pointer"), (dict(codes=None), "null pointer"),
    (dict(scales=None), "null pointer"), (dict(codes=ODD), "16-byte"), (dict(scales=ODD), "16-byte")]


@pytest.mark.parametrize("change,text", QUANT_CHANGES)
def test_mxfp4_conversion_refusals(lib, change, text):
    a = {**QUANT, **change}
    refused(lib, lib.pxs_quantize_mxfp4(*a.values()), text)
    refused(lib, lib.pxs_dequantize_mxfp4(a["codes"], a["scales"], a["rows"], a["channels"], a["dtype"], a["x"], a["ld"], None), text)


LINEAR = dict(x=P, xs=P, rows=4, cin=64, w=P, ws=P, bias=None, cout=32, act=0, dtype=0, y=P, stream=None)
SHARED = [
    (dict(rows=-1), "bad shape"), (dict(cin=0), "bad shape"), (dict(cout=0), "bad shape"), (dict(cin=2 ** 24 + 1), "2^24 inputs"),
    (dict(cout=2 ** 30 + 1), "2^30 outputs"), (dict(x=None), "null pointer"), (dict(xs=None), "null pointer"),
    (dict(w=None), "null pointer"), (dict(ws=None), "null pointer"), (dict(x=ODD), "16-byte"), (dict(xs=ODD), "16-byte"),
    (dict(w=ODD), "16-byte"), (dict(ws=ODD), "16-byte"), (dict(rows=2 ** 40, cin=1, cout=2 ** 20), "grid too large")]


@pytest.mark.parametrize("change,text", SHARED + [(dict(dtype=7), "bad dtype"), (dict(act=9), "bad activation"), (dict(y=None), "null pointer")])
def test_linear_mxfp4_refusals(lib, change, text):
    refused(lib, lib.pxs_linear_mxfp4(*{**LINEAR, **change}.values()), text)


@pytest.mark.parametrize("change,text", SHARED + [(dict(residual=None), "null pointer")])
def test_linear_mxfp4_residual_refusals(lib, change, text):
    base = dict(x=P, xs=P, rows=4, cin=64, w=P, ws=P, bias=None, cout=32)
    refused(lib, lib.pxs_linear_mxfp4_residual(*{**base, "residual": P, "stream": None, **change}.values()), text)
    gate = {**base, "coords": P, "bmod": P, "tmod": P, "offset": 0, "residual": P, "stream": None}
    refused(lib, lib.pxs_linear_mxfp4_gate_residual(*{**gate, **change}.values()), text)


@pytest.mark.parametrize("change,text", [(dict(offset=-1), "gate offset"), (dict(offset=161), "gate offset"),
                                         (dict(coords=None), "null pointer"), (dict(bmod=None), "null pointer"),
                                         (dict(tmod=None), "null pointer")])
def test_linear_mxfp4_gate_refusals(lib, change, text):
    gate = dict(x=P, xs=P, rows=4, cin=64, w=P, ws=P, bias=None, cout=32, coords=P, bmod=P, tmod=P, offset=0, residual=P,
                stream=None)
    refused(lib, lib.pxs_linear_mxfp4_gate_residual(*{**gate, **change}.values()), text)


def test_linear_mxfp4_tile(lib):
    tile = (C.c_int * 3)(7, 7, 7)
    assert lib.pxs_linear_mxfp4_tile(0, 64, 64, tile) == pxs.PXS_OK and list(tile) == [0, 0, 0]
    for args in ((-1, 64, 64, tile), (1, 0, 64, tile), (1, 64, 0, tile), (1, 2 ** 24 + 1, 64, tile), (1, 64, 2 ** 30 + 1, tile)):
        refused(lib, lib.pxs_linear_mxfp4_tile(*args), "bad shape")
    refused(lib, lib.pxs_linear_mxfp4_tile(1, 64, 64, None), "null pointer")


def test_mxfp4_of_nothing(lib):
    assert lib.pxs_quantize_mxfp4(*{**QUANT, "rows": 0, "x": None}.values()) == pxs.PXS_OK
    assert lib.pxs_dequantize_mxfp4(None, None, 0, 64, 0, None, 64, None) == pxs.PXS_OK
    assert lib.pxs_linear_mxfp4(*{**LINEAR, "rows": 0, "x": None}.values()) == pxs.PXS_OK


TREE = dict(dtype=1, q=P, ld_q=256, k=P, ld_k=128, v=P, ld_v=128, cu_q=P, parents=P, kc=P, ld_kc=128, vc=P, ld_vc=128,
            start=P, len=P, nseg=2, total_q=10, cache_rows=20, heads=4, kv=2, d=64, scale=0.125, cap=0.0, slopes=None,
            positions=None, o=P, ld_o=256, ws=P, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=5), "bad dtype"), (dict(heads=5), "multiple of kv_heads"), (dict(kv=0), "multiple of kv_heads"),
    (dict(heads=131072, kv=1), "65535"), (dict(d=0), "head_dim"), (dict(d=257), "head_dim"), (dict(scale=0.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(scale=3e38), "out of range"), (dict(cap=-1.0), "cap"), (dict(cap=math.inf), "cap"),
    (dict(cap=1e-44), "out of range"), (dict(slopes=P), "positions"), (dict(nseg=-1), "row counts"),
    (dict(total_q=-1), "row counts"), (dict(cache_rows=-1), "row counts"), (dict(cache_rows=2 ** 31 - 1023), "row counts"),
    (dict(total_q=2 ** 31 - 1024, heads=4, kv=2), "row counts"), (dict(ld_q=255), "row stride"), (dict(ld_k=127), "row stride"),
    (dict(ld_v=127), "row stride"), (dict(ld_kc=127), "row stride"), (dict(ld_vc=127), "row stride"), (dict(ld_o=255), "row stride"),
    (dict(q=None), "null pointer"), (dict(k=None), "null pointer"), (dict(v=None), "null pointer"), (dict(o=None), "null pointer"),
    (dict(kc=None), "null pointer"), (dict(vc=None), "null pointer"), (dict(cu_q=None), "null pointer"),
    (dict(parents=None), "null pointer"), (dict(start=None), "null pointer"), (dict(len=None), "null pointer"),
    (dict(ws=None), "null pointer"), (dict(ws=ODD), "256-byte aligned"),
    (dict(total_q=2 ** 31 - 1024, heads=65535, kv=65535, ld_q=2 ** 23, ld_k=2 ** 23, ld_v=2 ** 23, ld_kc=2 ** 23, ld_vc=2 ** 23,
          ld_o=2 ** 23), "grid too large")])
def test_tree_attention_refusals(lib, change, text):
    refused(lib, lib.pxs_tree_attention(*{**TREE, **change}.values()), text)


def test_tree_attention_of_nothing(lib):
    for change in (dict(nseg=0), dict(total_q=0)):
        assert lib.pxs_tree_attention(*{**TREE, **change}.values()) == pxs.PXS_OK


def test_tree_workspace_never_shrinks(lib):
    size = lib.pxs_tree_attention_workspace_bytes
    for heads, kv, d in ((1, 1, 64), (32, 8, 128), (16, 16, 64), (5, 5, 256)):
        last = 0
        for n in (0, 1, 2, 63, 64, 65, 1000, 10 ** 6):
            sizes = [size(n, rows, heads, kv, d) for rows in (0, 1, 10, 1000, 10 ** 6)]
            assert sizes == sorted(sizes) and sizes[-1] >= last
            last = sizes[-1]
