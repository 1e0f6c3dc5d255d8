"""One layer's step over drafted trees, as the operators are used together: the RMS norm into
8-bit rows, the 8-bit qkv product, q and k turned by their tokens' depths, attention of the trees
over the cache, the 4-bit output product, the norm that adds it to the residual, and a 4-bit MLP
whose second product is added as well.  Accepted tokens then join the cache.

Every stage is held to its own formula on the inputs it had (the tolerances of the stages' own
test files); the step is captured into graphs and replayed over caches that grow, and run on two
streams."""

import math

import numpy as np
import pytest
import torch

import pxs
from test_gpu_attention_scores import check as check_attn
from test_gpu_attention_tree import Batch
from test_gpu_linear_i8 import bounds as linear_bounds, check as check_linear, reference as reference_i8
from test_gpu_linear_mxfp4 import quantized as mx_quantized, reference as reference_mx
from test_gpu_rms_norm import U, LEAST, formula as norm_formula, near
from test_gpu_rope_positions import check as check_rope, turned

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, WIDTH, HIDDEN, EPS = 8, 2, 64, 512, 1370, 1e-6
TURNED, QKV = (HEADS + KV) * DIM, (HEADS + 2 * KV) * DIM
BF16 = torch.bfloat16
TREES = [([1], [0]), ([1], [700]), ([8, 5, 1, 0, 8], [300, 17, 0, 40, 1001]), ([200, 33], [130, 64])]


@pytest.fixture(scope="module")
def px():
    return pxs.Pxs()


def host(t):
    return t.cpu().numpy()


class Layer:
    """Weights quantized once, a batch with its cache, and the buffers a server keeps."""

    def __init__(self, px, q_len, k_len, seed):
        gen = torch.Generator("cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
        self.px, self.b = px, Batch(q_len, k_len, HEADS, KV, DIM, BF16, seed, cap=20.0, bias=True, gain=1.0)
        rows = self.rows = sum(q_len)
        self.g1, self.g2 = torch.exp(0.3 * rand(WIDTH)), torch.exp(0.3 * rand(WIDTH))
        self.wqkv, self.sqkv = px.quantize_rows(rand(QKV, WIDTH) / math.sqrt(WIDTH))
        self.bqkv, self.bout, self.bup, self.bdown = (0.1 * rand(n) for n in (QKV, WIDTH, HIDDEN, WIDTH))
        self.out, self.up, self.down = (px.quantize_mxfp4(rand(n, k) / math.sqrt(k))
                                        for n, k in ((WIDTH, HEADS * DIM), (HIDDEN, WIDTH), (WIDTH, HIDDEN)))
        self.freq = px.rope_frequencies(DIM, 10000.0, 4.0, 1024.0, 1.0, 32.0)
        empty = lambda n, dtype=BF16: torch.empty((rows, n), dtype=dtype, device="cuda")  # noqa: E731
        self.xq, self.xs = empty(WIDTH, torch.int8), torch.empty(rows, device="cuda")
        self.plain, self.attn, self.joined = empty(QKV), empty(HEADS * DIM), empty(WIDTH)
        self.normed, self.hidden = empty(WIDTH), empty(HIDDEN)
        self.a4, self.n4, self.h4 = (px.quantize_mxfp4(t.zero_()) for t in (self.attn, self.normed, self.hidden))
        self.ws = px.tree_attention_workspace(len(q_len), rows, HEADS, KV, DIM)
        self.residual0 = 2.0 * rand(rows, WIDTH)

    def __call__(self, residual):
        px, b = self.px, self.b
        px.rms_norm_i8(residual, EPS, self.g1, out=self.xq, scales=self.xs)
        px.linear_i8(self.xq, self.xs, self.wqkv, self.sqkv, self.bqkv, out=self.plain)
        b.qkv[:, TURNED:] = self.plain[:, TURNED:]
        px.rope_positions(self.plain[:, :TURNED], b.t_positions, self.freq, HEADS + KV, DIM, pxs.ROPE_HALF, out=b.qkv[:, :TURNED])
        b.run(px, out=self.attn, workspace=self.ws)
        px.quantize_mxfp4(self.attn, *self.a4)
        px.linear_mxfp4(*self.a4, *self.out, HEADS * DIM, self.bout, out=self.joined)
        px.rms_norm(self.joined, EPS, self.g2, residual, out=self.normed)
        px.quantize_mxfp4(self.normed, *self.n4)
        px.linear_mxfp4(*self.n4, *self.up, WIDTH, self.bup, pxs.ACT_SILU, out=self.hidden)
        px.quantize_mxfp4(self.hidden, *self.h4)
        px.linear_mxfp4_residual(*self.h4, *self.down, HIDDEN, self.bdown, residual)
        return residual

    def accept(self):
        """Each tree's first token, and a child of it where there is one, join the cache."""
        b, q0 = self.b, 0
        for i, n in enumerate(b.q_len):
            take = [0][:n] + [t for t in range(1, n) if b.parents[i][t] == 0][:1]
            for t in take:
                b.cache[b.start[i] + b.k_len[i]] = b.qkv[q0 + t, HEADS * DIM:]
                b.k_len[i] += 1
            q0 += n
        b.t_len.copy_(torch.tensor(b.k_len))
        b.t_positions.copy_(torch.tensor([b.k_len[i] + x for i, dep in enumerate(b.depth) for x in dep], dtype=torch.int32))


def check_mx(x, pair, weight, cin, bias):
    """-> (the product before the activation, its error bound) of the rows as they were quantized."""
    codes, scales = mx_quantized(x.double().cpu().numpy())
    np.testing.assert_array_equal(host(pair[0]), codes)
    np.testing.assert_array_equal(host(pair[1]), scales)
    return reference_mx((codes, scales), tuple(map(host, weight)), host(bias), cin)


def check_step(layer, before, after):
    b = layer.b
    _, _, q, scale = norm_formula(before, None, layer.g1, EPS)
    np.testing.assert_array_equal(host(layer.xq), q)
    near(layer.xs, scale, 3 * U * np.abs(scale) + LEAST)
    v, bound = reference_i8(host(layer.xq), host(layer.xs), host(layer.wqkv), host(layer.sqkv), host(layer.bqkv))
    check_linear(layer.plain, *linear_bounds(v, bound, "none", "bf16"), "qkv")
    want, size = turned(layer.plain[:, :TURNED].float().cpu().numpy(), host(b.t_positions), host(layer.freq), HEADS + KV, DIM, "half", 1.0)
    check_rope(b.qkv[:, :TURNED], want, size, True, "turned heads")
    check_attn(layer.attn, *b.want(), "attention")
    v, bound = check_mx(layer.attn, layer.a4, layer.out, HEADS * DIM, layer.bout)
    check_linear(layer.joined, *linear_bounds(v, bound, "none", "bf16"), "output product")
    middle, y, _, _ = norm_formula(layer.joined, before, layer.g2, EPS)
    tol = 3 * U * np.abs(y) + LEAST
    near(layer.normed, y, tol + 2.0 ** -8 * (np.abs(y) + tol) + 2.0 ** -134)
    v, bound = check_mx(layer.normed, layer.n4, layer.up, WIDTH, layer.bup)
    check_linear(layer.hidden, *linear_bounds(v, bound, "silu", "bf16"), "up")
    v, bound = check_mx(layer.hidden, layer.h4, layer.down, HIDDEN, layer.bdown)
    want = middle.double().numpy() + v
    check_linear(after, want, bound + U * (np.abs(want) + bound) + 1e-38, "residual")


@pytest.mark.parametrize("q_len,k_len", TREES)
def test_step_stage_by_stage(px, q_len, k_len):
    layer = Layer(px, q_len, list(k_len), 51)
    for _ in range(2):  # the second over the cache that the first's accepted tokens have joined
        after = layer(layer.residual0.clone())
        check_step(layer, layer.residual0, after)
        layer.accept()


@pytest.mark.parametrize("q_len,k_len", TREES[1:])
def test_step_in_graphs(px, q_len, k_len):
    """Captured twice and replayed with eager steps between, over one workspace: the cache grows, its rows
    move, and the residual changes between the replays."""
    layer = Layer(px, q_len, list(k_len), 52)
    outs = [layer.residual0.clone() for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(outs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            layer(out)
        graphs.append(g)
    layer.b.cache.nan_to_num_(0.5)
    rows = layer.b.cache.shape[0]
    for turn in range(4):
        now = torch.randn(outs[0].shape, device="cuda", generator=torch.Generator("cuda").manual_seed(60 + turn))
        if turn < 2:
            layer.accept()
        else:  # every length from nothing to the whole cache, wherever it starts
            lens = [(0, 1, 128, rows, rows // 2)[(turn + i) % 5] for i in range(len(q_len))]
            layer.b.t_len.copy_(torch.tensor([min(n, rows) for n in lens]))
            layer.b.t_start.copy_(torch.tensor([(rows - min(n, rows)) // 2 for n in lens]))
        want = layer(now.clone())
        assert torch.isfinite(want).all()
        for g, out in zip(graphs, outs):
            out.copy_(now)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), f"replay {turn}"
            layer(now.clone())  # eager work between


def test_two_streams_at_once(px):
    """Two layers with buffers of their own, each on its stream, meet their results alone."""
    layers = [Layer(px, q, list(k), 53 + i) for i, (q, k) in enumerate(TREES[2:])]
    alone = [layer(layer.residual0.clone()) for layer in layers]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in layers], [layer.residual0.clone() for layer in layers]
    torch.cuda.synchronize()
    for _ in range(3):
        for layer, stream, out in zip(layers, streams, outs):
            with torch.cuda.stream(stream):
                out.copy_(layer.residual0)
                layer(out)
        torch.cuda.synchronize()
        for out, want in zip(outs, alone):
            assert torch.equal(out, want)


def test_padded_batch(px):
    """Rows behind the last tree: the norms and products take them, the attention leaves theirs as they were."""
    q_len, k_len, spare = [8, 5], [300, 17], 3
    b = Batch(q_len, k_len, HEADS, KV, DIM, BF16, 54, spare=spare)
    rows = sum(q_len)
    attn = torch.full((rows + spare, HEADS * DIM), 0.25, dtype=BF16, device="cuda")
    px.tree_attention(*(t.nan_to_num(1.0) for t in (b.q, b.k, b.v)), b.cu, b.t_parents, b.kc, b.vc, b.t_start, b.t_len,
                      HEADS, KV, DIM, b.scale, out=attn)
    check_attn(attn[:rows], *b.want(), "attention")
    assert (attn[rows:] == 0.25).all()
    codes, scales = px.quantize_mxfp4(attn)
    want_codes, want_scales = mx_quantized(attn.double().cpu().numpy())
    np.testing.assert_array_equal(host(codes), want_codes)
    np.testing.assert_array_equal(host(scales), want_scales)


def test_first_calls_inside_a_capture(px):
    """Kernels that need more than 64 KB of LDS, called for the first time under capture."""
    small = Batch([40, 3], [200, 500], 2, 1, 256, torch.float32, 55)
    wide = Batch([64, 3], [200, 500], 8, 2, 128, BF16, 56)
    x, w = torch.randn(600, 1024, device="cuda"), torch.randn(1024, 1024, device="cuda")
    xq, wq = px.quantize_mxfp4(x), px.quantize_mxfp4(w)
    outs = [torch.zeros((t.rows, t.heads * t.d), dtype=t.dtype, device="cuda") for t in (small, wide)]
    y = torch.zeros((600, 1024), device="cuda")
    spaces = [px.tree_attention_workspace(2, t.rows, t.heads, t.kv, t.d) for t in (small, wide)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for t, out, ws in zip((small, wide), outs, spaces):
            t.run(px, out=out, workspace=ws)
        px.linear_mxfp4(*xq, *wq, 1024, out=y)
    for _ in range(3):
        for t in (*outs, y):
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        for t, out in zip((small, wide), outs):
            check_attn(out, *t.want(), "captured")
        v, bound = reference_mx(tuple(map(host, xq)), tuple(map(host, wq)), None, 1024)
        check_linear(y, v, bound, "captured product")
