"""The 8-bit linears, rotary positions and scored attention together, as one
attention layer over token sequences uses them: quantized activations through
the qkv product, q and k turned in place in the packed projection, attention
over a cache with shared key/value heads, quantization, and the output product
added to the residual.

Every stage is held to its own formula on the inputs it had (the tolerances of
the stages' own test files); the layer is run whole and token by token, captured
into graphs and replayed, and on other streams."""

import math

import numpy as np
import pytest
import torch

import pxs
from test_gpu_attention_scores import bounds, check as check_attn, formula
from test_gpu_linear_i8 import bounds as linear_bounds, check as check_linear, quantized, reference
from test_gpu_rope_positions import check as check_rope, turned

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, WIDTH = 8, 2, 64, 512
QKV = (HEADS + 2 * KV) * DIM


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


class Layer:
    """Weights quantized once, and the buffers a server keeps."""

    def __init__(self, px, seed, rows, cache_rows, nseg):
        gen = torch.Generator("cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
        self.px = px
        self.wqkv, self.sqkv = px.quantize_rows(rand(QKV, WIDTH) / math.sqrt(WIDTH))
        self.wout, self.sout = px.quantize_rows(rand(WIDTH, HEADS * DIM) / math.sqrt(HEADS * DIM))
        self.bqkv, self.bout = 0.1 * rand(QKV), 0.1 * rand(WIDTH)
        self.freq = px.rope_frequencies(DIM, 10000.0, 4.0, 1024.0, 1.0, 32.0)
        self.slopes = torch.exp2(-torch.arange(1, HEADS + 1, device="cuda", dtype=torch.float32))
        self.k_cache = torch.zeros((cache_rows, KV * DIM), dtype=torch.bfloat16, device="cuda")
        self.v_cache = torch.zeros_like(self.k_cache)
        self.xq = torch.empty((rows, WIDTH), dtype=torch.int8, device="cuda")
        self.xs = torch.empty(rows, device="cuda")
        self.qkv = torch.empty((rows, QKV), dtype=torch.bfloat16, device="cuda")
        self.attn = torch.empty((rows, HEADS * DIM), dtype=torch.bfloat16, device="cuda")
        self.aq = torch.empty((rows, HEADS * DIM), dtype=torch.int8, device="cuda")
        self.as_ = torch.empty(rows, device="cuda")
        self.ws = px.attention_scores_workspace(nseg, rows, cache_rows, HEADS, KV, DIM)

    def __call__(self, x, positions, slots, cu_q, cu_k, residual, total_k):
        px = self.px
        px.quantize_rows(x, out=self.xq, scales=self.xs)
        px.linear_i8(self.xq, self.xs, self.wqkv, self.sqkv, self.bqkv, out=self.qkv)
        turn = self.qkv[:, :(HEADS + KV) * DIM]
        px.rope_positions(turn, positions, self.freq, HEADS + KV, DIM, pxs.ROPE_HALF, out=turn)
        self.k_cache[slots] = self.qkv[:, HEADS * DIM:(HEADS + KV) * DIM]
        self.v_cache[slots] = self.qkv[:, (HEADS + KV) * DIM:]
        px.varlen_attention_scores(self.qkv[:, :HEADS * DIM], self.k_cache[:total_k], self.v_cache[:total_k], cu_q, cu_k,
                                   HEADS, KV, DIM, 1.0 / math.sqrt(DIM), cap=20.0, slopes=self.slopes, causal=True,
                                   out=self.attn, workspace=self.ws)
        px.quantize_rows(self.attn, out=self.aq, scales=self.as_)
        px.linear_i8_residual(self.aq, self.as_, self.wout, self.sout, self.bout, residual)
        return residual


def prompt(lens, seed):
    rows = sum(lens)
    gen = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((rows, WIDTH), device="cuda", generator=gen).bfloat16()
    residual = torch.randn((rows, WIDTH), device="cuda", generator=gen)
    positions = torch.cat([torch.arange(n, device="cuda") for n in lens]).to(torch.int32)
    return x, residual, positions, torch.arange(rows, device="cuda")


@pytest.mark.parametrize("lens", [[1], [200, 37, 1], [513, 129]])
def test_layer_stage_by_stage(px, lens):
    rows = sum(lens)
    layer = Layer(px, 21, rows, rows, len(lens))
    x, residual, positions, slots = prompt(lens, 22)
    before = residual.clone()
    host = lambda t: t.cpu().numpy()  # noqa: E731
    # the projection before its heads are turned
    q8, s8 = px.quantize_rows(x)
    plain = px.linear_i8(q8, s8, layer.wqkv, layer.sqkv, layer.bqkv)
    layer(x, positions, slots, bounds(lens), bounds(lens), residual, rows)
    want_q, want_s = quantized(x.float().cpu().numpy())
    np.testing.assert_array_equal(host(layer.xq), want_q)
    np.testing.assert_array_equal(host(layer.xs), want_s)
    v, bound = reference(want_q, want_s, host(layer.wqkv), host(layer.sqkv), host(layer.bqkv))
    check_linear(plain, *linear_bounds(v, bound, "none", "bf16"), "qkv")
    n = (HEADS + KV) * DIM
    want, size = turned(plain[:, :n].float().cpu().numpy(), host(positions), host(layer.freq), HEADS + KV, DIM, "half", 1.0)
    check_rope(layer.qkv[:, :n], want, size, True, "turned heads")
    assert torch.equal(layer.qkv[:, n:], plain[:, n:])
    want, tol = formula(layer.qkv[:, :HEADS * DIM], layer.k_cache, layer.v_cache, lens, lens, HEADS, KV, DIM,
                        1.0 / math.sqrt(DIM), 20.0, layer.slopes, True)
    check_attn(layer.attn, want, tol, "attention")
    want_q, want_s = quantized(layer.attn.float().cpu().numpy())
    np.testing.assert_array_equal(host(layer.aq), want_q)
    v, bound = reference(want_q, want_s, host(layer.wout), host(layer.sout), host(layer.bout))
    want = host(before).astype(np.float64) + v
    check_linear(residual, want, bound + 2.0 ** -24 * np.abs(want) + 1e-38, "residual")


def test_token_by_token_meets_the_whole_prompt(px):
    """Single tokens over the cache that the prompt left: the same attention rows, to
    the two calls' roundings."""
    length = 150
    whole = Layer(px, 23, length, length, 1)
    x, residual, positions, slots = prompt([length], 24)
    whole(x, positions, slots, bounds([length]), bounds([length]), residual.clone(), length)
    one = Layer(px, 23, 1, length, 1)
    for t in (0, 1, 63, 64, 100, length - 1):
        one.k_cache[:t] = whole.k_cache[:t]
        one.v_cache[:t] = whole.v_cache[:t]
        one(x[t:t + 1], positions[t:t + 1], slots[t:t + 1], bounds([1]), bounds([t + 1]), residual[t:t + 1].clone(), t + 1)
        # everything before the attention is row by row, and equal
        assert torch.equal(one.qkv, whole.qkv[t:t + 1])
        want, tol = formula(one.qkv[:, :HEADS * DIM], whole.k_cache[:t + 1], whole.v_cache[:t + 1], [1], [t + 1], HEADS, KV,
                            DIM, 1.0 / math.sqrt(DIM), 20.0, whole.slopes, True)
        check_attn(one.attn, want, tol, f"token {t}")
        check_attn(whole.attn[t:t + 1], want, tol, f"row {t} of the prompt")


@pytest.mark.parametrize("lens,cache", [([300, 65], None), ([1, 1, 1], [700, 1, 90])])
def test_layer_in_a_graph(px, lens, cache):
    """Captured and replayed with new inputs between replays, eager work around them;
    two graphs share the workspace and buffers."""
    rows, k_lens = sum(lens), cache or lens
    total = sum(k_lens)
    layer = Layer(px, 25, rows, total, len(lens))
    layer.k_cache.normal_(generator=torch.Generator("cuda").manual_seed(1))
    layer.v_cache.normal_(generator=torch.Generator("cuda").manual_seed(2))
    ends = torch.cumsum(torch.tensor(k_lens, device="cuda"), 0)
    x, residual, positions, slots = prompt(lens, 26)
    if cache:
        slots, positions = ends - 1, (torch.tensor(k_lens, device="cuda") - 1).to(torch.int32)
    cu_q, cu_k = bounds(lens), bounds(k_lens)
    out_a, out_b = residual.clone(), residual.clone()
    run = lambda out: layer(x, positions, slots, cu_q, cu_k, out, total)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(out_a)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for out in (out_a, out_b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(out)
        graphs.append(g)
    for turn in range(4):
        x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(30 + turn)))
        want = run(residual.clone())
        for g, out in zip(graphs, (out_a, out_b)):
            out.copy_(residual)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), f"replay {turn}"
            residual.add_(0.0)  # eager work between


def test_two_streams_at_once(px):
    """Two layers with buffers of their own, each on its stream, meet their results alone."""
    layers = [Layer(px, 27 + i, n, n, 1) for i, n in enumerate((700, 333))]
    data = [prompt([n], 40 + i) for i, n in enumerate((700, 333))]
    cus = [bounds([n]) for n in (700, 333)]
    alone = [layer(x, pos, slots, cu, cu, res.clone(), len(x)).clone()
             for layer, (x, res, pos, slots), cu in zip(layers, data, cus)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    outs = [res.clone() for _, res, _, _ in data]
    torch.cuda.synchronize()
    for _ in range(3):
        for layer, stream, (x, res, pos, slots), cu, out in zip(layers, streams, data, cus, outs):
            with torch.cuda.stream(stream):
                out.copy_(res)
                layer(x, pos, slots, cu, cu, out, len(x))
        torch.cuda.synchronize()
        for out, want in zip(outs, alone):
            assert torch.equal(out, want)


def test_first_calls_inside_a_capture(px):
    """Kernels that need more than 64 KB of LDS, called for the first time under capture."""
    n, d = 40, 256
    q, k, v = (torch.randn((n, d), device="cuda", generator=torch.Generator("cuda").manual_seed(s)) for s in (1, 2, 3))
    cu, o = bounds([n]), torch.zeros((n, d), device="cuda")
    ws = px.attention_scores_workspace(1, n, n, 1, 1, d)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        px.varlen_attention_scores(q, k, v, cu, cu, 1, 1, d, 0.05, causal=True, out=o, workspace=ws)
    for _ in range(2):
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        want, tol = formula(q, k, v, [n], [n], 1, 1, d, 0.05, causal=True)
        check_attn(o, want, tol, "captured")


def test_padded_batch(px):
    """Rows of q, k and v past the last segment: q's are left out, and o's as they were."""
    for lens, heads, kv, d, dtype in (([5, 9], 4, 2, 64, torch.bfloat16), ([1, 1], 4, 2, 64, torch.bfloat16),
                                      ([200, 100], 4, 2, 72, torch.bfloat16), ([1, 2], 2, 2, 64, torch.float32)):
        n = sum(lens)
        gen = torch.Generator("cuda").manual_seed(50)
        q = torch.randn((n + 7, heads * d), device="cuda", generator=gen).to(dtype)
        k, v = (torch.randn((3000 + n, kv * d), device="cuda", generator=gen).to(dtype) for _ in range(2))
        q[n:], k[n + 2000:], v[n + 2000:] = math.nan, math.nan, math.nan
        k_lens = [lens[0] + 1300, lens[1] + 700]
        o = torch.full((n + 7, heads * d), 3.0, device="cuda").to(dtype)
        px.varlen_attention_scores(q, k, v, bounds(lens), bounds(k_lens), heads, kv, d, 0.1, causal=True, out=o)
        want, tol = formula(q[:n], k[:sum(k_lens)], v[:sum(k_lens)], lens, k_lens, heads, kv, d, 0.1, causal=True)
        check_attn(o[:n], want, tol, f"{lens}")
        assert (o[n:] == 3.0).all()


def test_bounds_past_the_rows_stay_inside(px):
    """cu_seqlens that point past the rows given are cut to them (the caller's mistake, but no
    read or write leaves the tensors): the rows that do exist are right."""
    q, k, v = (torch.randn((64, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(s)).bfloat16() for s in (1, 2, 3))
    good = px.varlen_attention_scores(q, k, v, bounds([64]), bounds([64]), 1, 1, 64, 0.1)
    wide = torch.tensor([0, 100], device="cuda")
    for segs in (1, 70):
        cu = torch.cat([wide, wide.new_full((segs - 1,), 100)])
        assert torch.equal(px.varlen_attention_scores(q, k, v, cu, cu, 1, 1, 64, 0.1), good)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("segs", [3, 70])
def test_bounds_that_fall_stay_inside(px, segs, dtype):
    """Segments that overlap, or whose bounds fall: what they compute is undefined, but rows around the
    tensors' stay as they were, and a call that follows is right."""
    rows, keys, d = 48, 3000, 64
    gen = torch.Generator("cuda").manual_seed(51)
    q = torch.randn((rows, d), device="cuda", generator=gen).to(dtype)
    k, v = (torch.randn((keys, d), device="cuda", generator=gen).to(dtype) for _ in range(2))
    around = torch.full((rows + 64, d), 3.0, device="cuda").to(dtype)
    o = around[32:32 + rows]
    good = px.varlen_attention_scores(q, k, v, bounds([rows]), bounds([keys]), 1, 1, d, 0.1)
    for cu_q, cu_k in (([0, 40, 8, rows], [0, keys, 100, keys]), ([0, 20, 48, 10], [0, keys, 0, keys]),
                       ([5, 2, 48, 48], [7, 3, keys, 9]), ([0, -9, 60, 20], [-5, keys + 9, 0, keys])):
        fill = [cu_q[-1]] * (segs - 3), [cu_k[-1]] * (segs - 3)
        cq, ck = (torch.tensor(c + f, device="cuda") for c, f in zip((cu_q, cu_k), fill))
        px.varlen_attention_scores(q, k, v, cq, ck, 1, 1, d, 0.1, causal=True, out=o)
        assert (around[:32] == 3.0).all() and (around[32 + rows:] == 3.0).all()
    assert torch.equal(px.varlen_attention_scores(q, k, v, bounds([rows]), bounds([keys]), 1, 1, d, 0.1), good)


def test_wrong_tensors_are_refused(px):
    x = torch.zeros((4, 64), device="cuda", dtype=torch.bfloat16)
    q, s = px.quantize_rows(x)
    w, ws = px.quantize_rows(torch.ones((32, 64), device="cuda"))
    for call in (lambda: px.quantize_rows(x.cpu()), lambda: px.quantize_rows(x.t()[:, :4]),
                 lambda: px.quantize_rows(x, out=q[:2]), lambda: px.linear_i8(q, s[:2], w, ws),
                 lambda: px.linear_i8(q, s, w, ws.double()), lambda: px.linear_i8(q, s, w[:, :32], ws),
                 lambda: px.linear_i8(q, s, w, ws, torch.ones(31, device="cuda")),
                 lambda: px.linear_i8(x, s, w, ws),
                 lambda: px.linear_i8_residual(q, s, w, ws, None, torch.zeros((4, 32), device="cuda").bfloat16()),
                 lambda: px.rope_positions(x, torch.zeros(4, device="cuda"), px.rope_frequencies(64), 1, 64),
                 lambda: px.rope_positions(x, torch.zeros(3, device="cuda", dtype=torch.int32), px.rope_frequencies(64), 1, 64),
                 lambda: px.rope_positions(x, torch.zeros(4, device="cuda", dtype=torch.int32), px.rope_frequencies(66), 1, 64),
                 lambda: px.varlen_attention_scores(x, x, x[:2], bounds([4]), bounds([4]), 1, 1, 64, 0.1),
                 lambda: px.varlen_attention_scores(x, x, x, bounds([4]), bounds([4]).int(), 1, 1, 64, 0.1),
                 lambda: px.varlen_attention_scores(x, x, x, bounds([4]), bounds([4]), 1, 1, 64, 0.1, slopes=torch.ones(2, device="cuda")),
                 lambda: px.varlen_attention_scores(x, x, x, bounds([4]), bounds([4]), 1, 1, 64, 0.1,
                                                    workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(pxs.PxsError):
            call()
