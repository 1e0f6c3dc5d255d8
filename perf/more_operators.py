"""What a served token model needs around its 8-bit linears and its scored
attention: what these are measured on.

Three kinds of case:
  norm  the residual's addition and the root-mean-square norm of its rows, with
        rows of 8-bit integers and a scale each (the 8-bit linears' input), or
        rows of the call's type;
  mx    microscaled 4-bit floating point (blocks of 32 values of two exponent
        bits and one of mantissa under a power of two): activations quantized,
        then the product with 4-bit weights, bias and activation; or values
        quantized and read back;
  tree  attention of a tree of drafted tokens over a cache: a token sees its
        sequence's cached keys, its ancestors in the tree and itself.

`prepare` makes what a caller holds before the call, `run` is one call (in
plain torch, or through the Python binding where `own` is set), `work` the
bytes and operations the call cannot do without, `exact` its outputs in 64
bits.  Widths, head counts and lengths are those of the flow model's blocks
(width 1024, MLP 4096, 16 heads of 64, 1,370 context tokens, up to 42k rows) or
generic.
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
ACTS = {"none": 0, "gelu": 1, "silu": 2}
EPS = 1e-6


# ---- cases -----------------------------------------------------------------

def listed():
    return [
        # One new token's row on its way into the first 8-bit linear of a block.
        dict(name="norm_token", kind="norm", x="bf16", residual="f32", rows=1, channels=1024, out="i8"),
        # The same at the flow model's largest voxel count.
        dict(name="norm_42k", kind="norm", x="bf16", residual="f32", rows=42017, channels=1024, out="i8"),
        # A residual in 16 bits, odd width (no whole 16-byte pieces), rows in the call's type.
        dict(name="norm_odd", kind="norm", x="bf16", residual="bf16", rows=4739, channels=1370, out="y"),
        # One new token through the first MLP linear of a block.
        dict(name="mx_token", kind="mx", dtype="bf16", rows=1, cin=1024, cout=4096, act="gelu"),
        # An image's 1,370 tokens through the same linear.
        dict(name="mx_mlp_1370", kind="mx", dtype="bf16", rows=1370, cin=1024, cout=4096, act="gelu"),
        # A long prompt through a wide model's linear: the product is most of it.
        dict(name="mx_wide", kind="mx", dtype="bf16", rows=8192, cin=8192, cout=4096, act="none"),
        # Odd sizes throughout, fp32 in and out: the last block of a row holds 26 values.
        dict(name="mx_odd_f32", kind="mx", dtype="f32", rows=4739, cin=1370, cout=1021, act="silu"),
        # An MLP's weights quantized when the model is loaded, and read back to be looked at.
        dict(name="mx_weights", kind="mxq", dtype="f32", rows=4096, cin=4096),
        # One sequence, a small tree over a short cache, every head its own keys.
        dict(name="tree_one", kind="tree", dtype="bf16", q="12", k="1501", heads=16, kv_heads=16, head_dim=64,
             cap=0.0, bias=0),
        # A batch of ragged caches with a few drafted tokens each.
        dict(name="tree_ragged", kind="tree", dtype="bf16", q="8,8,8,5,8,8,1,8",
             k="40001,32768,20480,9999,4739,1370,17,0", heads=32, kv_heads=8, head_dim=128, cap=0.0, bias=0),
        # Wide trees over prompts of equal size, capped scores.
        dict(name="tree_wide", kind="tree", dtype="bf16", q="64,64,61,64,64,64,64,50",
             k="8192,8192,8192,8192,8192,8192,8192,8192", heads=32, kv_heads=8, head_dim=128, cap=50.0, bias=0),
        # fp32, everything at once.
        dict(name="tree_f32", kind="tree", dtype="f32", q="37,100", k="2370,517", heads=16, kv_heads=8, head_dim=64,
             cap=20.0, bias=1),
    ]


def draw(rng: random.Random):
    """One more case of the listed kinds, over the whole range of sizes."""

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["norm", "mx", "mx", "mxq", "tree", "tree"])
    if kind == "norm":
        channels = rng.choice([rng.randint(17, 500), 1024, 1370, rng.randint(500, 4096), 4096, 8192])
        return dict(kind=kind, x=rng.choice(["f32", "bf16", "bf16"]), residual=rng.choice(["f32", "f32", "bf16", "none"]),
                    rows=log(1, 42017 * 1024 // max(channels, 1024)), channels=channels, out=rng.choice(["i8", "i8", "y"]))
    if kind == "mx":
        cin = rng.choice([rng.randint(33, 500), 1024, 1370, rng.randint(500, 4096), 4096])
        cout = rng.choice([rng.randint(8, 300), 1024, 1021, rng.randint(300, 4096), 4096])
        most = 8192 * 8192 * 4096 // (cin * cout)
        return dict(kind=kind, dtype=rng.choice(["f32", "bf16", "bf16"]), rows=log(1, min(42017, most)),
                    cin=cin, cout=cout, act=rng.choice(["none", "gelu", "silu"]))
    if kind == "mxq":
        cin = rng.choice([rng.randint(33, 500), 1024, 1370, 4096])
        return dict(kind=kind, dtype=rng.choice(["f32", "bf16"]), rows=log(1, 4096 * 4096 // cin), cin=cin)
    dtype = rng.choice(["f32", "bf16", "bf16", "bf16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    items = rng.randint(1, 8)
    width = rng.choice([4, 12, 30, 64])
    top = 8000 if dtype == "f32" or width > 12 else 30000
    return dict(kind=kind, dtype=dtype, q=",".join(str(rng.randint(1, width)) for _ in range(items)),
                k=",".join(str(log(1, top) - 1) for _ in range(items)), heads=kv_heads * rng.choice([1, 2, 3, 4]),
                kv_heads=kv_heads, head_dim=rng.choice([64, 64, 128, 128, 80, 96]),
                cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.choice([0, 0, 1]))


def _ints(text):
    return [int(n) for n in text.split(",")]


def _starts(lengths, room=0):
    return [sum(n + room for n in lengths[:i]) for i in range(len(lengths) + 1)]


# ---- inputs -----------------------------------------------------------------

class _State(dict):
    __getattr__ = dict.__getitem__


@functools.lru_cache(maxsize=1)
def _px():
    folder = str(Path(__file__).resolve().parents[1] / "pixal3d.cpp_amd" / "python")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import pxs
    return pxs.Pxs()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    s = _State(case=case)

    def tokens(rows, channels):
        # Tokens of different size, a few channels an order larger than the rest.
        channel = torch.exp(0.5 * rand(channels))
        channel[torch.randint(0, channels, (max(channels // 128, 1),), device="cuda", generator=gen)] *= 10.0
        return rand(rows, channels) * channel * torch.exp(0.3 * rand(rows, 1))

    if case["kind"] == "norm":
        rows, channels = case["rows"], case["channels"]
        s.x = tokens(rows, channels).to(DTYPES[case["x"]])
        s.gamma = torch.exp(0.2 * rand(channels))
        s.residual = s.residual_out = None
        if case["residual"] != "none":
            s.residual = (4.0 * tokens(rows, channels)).to(DTYPES[case["residual"]])
            s.residual_out = torch.empty_like(s.residual)
        if case["out"] == "i8":
            s.q = torch.empty((rows, channels), dtype=torch.int8, device="cuda")
            s.scales = torch.empty(rows, dtype=torch.float32, device="cuda")
        else:
            s.y = torch.empty((rows, channels), dtype=DTYPES[case["x"]], device="cuda")
    elif case["kind"] == "mx":
        rows, cin, cout = case["rows"], case["cin"], case["cout"]
        s.x = tokens(rows, cin).to(DTYPES[case["dtype"]])
        # Weights quantized once, when the model was loaded.
        w = rand(cout, cin) * (torch.exp(0.3 * rand(cout, 1)) / math.sqrt(cin))
        s.w, s.w_scales = _pack(*_quantize(w))
        s.bias = 0.1 * rand(cout)
        s.y = torch.empty((rows, cout), dtype=DTYPES[case["dtype"]], device="cuda")
        s.xq, s.x_scales = [torch.empty((rows, t.shape[1]), dtype=torch.uint8, device="cuda") for t in (s.w, s.w_scales)]
    elif case["kind"] == "mxq":
        rows, cin = case["rows"], case["cin"]
        s.x = (rand(rows, cin) * (torch.exp(0.3 * rand(rows, 1)) / math.sqrt(cin))).to(DTYPES[case["dtype"]])
        s.y = torch.empty_like(s.x)
    else:
        q_len, k_len = _ints(case["q"]), _ints(case["k"])
        heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        dtype = DTYPES[case["dtype"]]
        # Scores of a few units, as normalised q and k with learned gains give; the drafted
        # tokens' q, k and v are columns of one projection.
        qkv = rand(sum(q_len), (heads + 2 * kv) * d)
        qkv[:, :(heads + kv) * d] *= 2.0
        s.qkv = qkv.to(dtype)
        s.q, s.k, s.v = s.qkv[:, :heads * d], s.qkv[:, heads * d:(heads + kv) * d], s.qkv[:, (heads + kv) * d:]
        # Each sequence's cache has room for 64 more rows.
        start = _starts(k_len, 64)
        cache = rand(start[-1], 2 * kv * d)
        cache[:, :kv * d] *= 2.0
        s.cache = cache.to(dtype)
        s.k_cache, s.v_cache = s.cache[:, :kv * d], s.cache[:, kv * d:]
        device = dict(dtype=torch.int64, device="cuda")
        s.cu_q = torch.tensor(_starts(q_len), **device)
        s.cache_start, s.cache_len = torch.tensor(start[:-1], **device), torch.tensor(k_len, **device)
        # A tree grows from the last accepted token, each token from one of the newer ones.
        host = random.Random(seed)
        parents = [-1 if t == 0 else host.randint((t - 1) // 3, t - 1) for n in q_len for t in range(n)]
        depth = []
        for n, first in zip(q_len, _starts(q_len)):
            for t in range(n):
                depth.append(0 if t == 0 else 1 + depth[first + parents[first + t]])
        s.parents = torch.tensor(parents, dtype=torch.int32, device="cuda")
        s.positions = torch.tensor(depth, dtype=torch.int32, device="cuda") + \
            s.cache_len.to(torch.int32).repeat_interleave(torch.tensor(q_len, device="cuda"))
        s.slopes = None
        if case["bias"]:
            s.slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)
        s.scale = 1.0 / math.sqrt(d)
        s.o = torch.empty((sum(q_len), heads * d), dtype=dtype, device="cuda")
    return s


def _quantize(x):
    """Blocks of 32 of a row: (values in units of the block's scale [rows, blocks, 32], the scale's
    exponent [rows, blocks]).  The largest magnitude's exponent less 2; ties to even; past 6, 6."""
    rows, channels = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -channels % 32)).reshape(rows, -1, 32)
    exponent = (torch.frexp(x.abs().amax(2)).exponent - 3).clamp(-127, 125)
    exponent = torch.where((x == 0).all(2), -127, exponent)
    u = torch.ldexp(x, -exponent[:, :, None])
    m = u.abs()
    m = torch.where(m < 2.0, torch.round(m * 2.0) * 0.5, torch.where(m < 4.0, torch.round(m), torch.round(m * 0.5) * 2.0))
    return torch.copysign(m.clamp_max(6.0), u), exponent


def _pack(values, exponent):
    """The bytes of quantized blocks: two codes a byte, the earlier in the low half, and a row's scales in
    whole 16 bytes."""
    m = values.abs()
    code = torch.where(m < 2.0, m * 2.0, torch.where(m < 4.0, m + 2.0, m * 0.5 + 4.0)).to(torch.uint8)
    code = code | (torch.signbit(values).to(torch.uint8) << 3)
    code = code.flatten(1)
    scales = torch.nn.functional.pad((exponent + 127).to(torch.uint8), (0, -exponent.shape[1] % 16), value=127)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scales.contiguous()


def _unpack(codes, scales, channels):
    """The values that the bytes stand for, in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], dim=2).flatten(1).to(torch.int32)
    m = code & 7
    value = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2.0, m * 2.0 - 8.0))
    value = torch.where(code >= 8, -value, value).reshape(codes.shape[0], -1, 32)
    exponent = scales[:, :value.shape[1]].to(torch.int32) - 127
    return torch.ldexp(value, exponent[:, :, None]).flatten(1)[:, :channels].contiguous()


# ---- one call ------------------------------------------------------------------

def run(s):
    kind = s.case["kind"]
    if own:
        return {"norm": _own_norm, "mx": _own_mx, "mxq": _own_mxq, "tree": _own_tree}[kind](s)
    return {"norm": _norm, "mx": _mx, "mxq": _mxq, "tree": _tree}[kind](s)


def _own_norm(s):
    if s.case["out"] == "i8":
        _px().rms_norm_i8(s.x, EPS, s.gamma, s.residual, s.residual_out, out=s.q, scales=s.scales)
        return {"q": s.q, "scales": s.scales, "residual": s.residual_out}
    _px().rms_norm(s.x, EPS, s.gamma, s.residual, s.residual_out, out=s.y)
    return {"y": s.y, "residual": s.residual_out}


def _own_mx(s):
    _px().quantize_mxfp4(s.x, out=s.xq, scales=s.x_scales)
    return _px().linear_mxfp4(s.xq, s.x_scales, s.w, s.w_scales, s.case["cin"], s.bias, ACTS[s.case["act"]], out=s.y)


def _own_mxq(s):
    codes, scales = _px().quantize_mxfp4(s.x)
    return _px().dequantize_mxfp4(codes, scales, s.case["cin"], out=s.y)


def _own_tree(s):
    c = s.case
    if "workspace" not in s:  # kept with the model's other buffers
        s["workspace"] = _px().tree_attention_workspace(s.cu_q.numel() - 1, s.q.shape[0], c["heads"], c["kv_heads"],
                                                        c["head_dim"], device="cuda")
    return _px().tree_attention(s.q, s.k, s.v, s.cu_q, s.parents, s.k_cache, s.v_cache, s.cache_start, s.cache_len,
                                c["heads"], c["kv_heads"], c["head_dim"], s.scale, cap=c["cap"], slopes=s.slopes,
                                positions=s.positions if c["bias"] else None, out=s.o, workspace=s.workspace)


def _norm(s):
    h = s.x.float()
    stored = None
    if s.residual is not None:
        stored = (s.residual.float() + h).to(s.residual.dtype)
        h = stored.float()
    inv = torch.rsqrt((h.double() * h.double()).mean(1) + EPS).float()
    t = h * s.gamma
    if s.case["out"] == "y":
        return {"y": (t * inv[:, None]).to(s.x.dtype), "residual": stored}
    # 8-bit rows of h * gamma, whose scale then takes the norm's factor; divisions of
    # tensors, each rounded once (by a number, torch multiplies with its inverse).
    most = t.abs().amax(1)
    live = most >= 2.0 ** -100
    top = torch.full_like(most, 127.0)
    per = torch.where(live, top / most.clamp_min(2.0 ** -100), torch.zeros_like(most))
    scales = torch.where(live, most / top, torch.zeros_like(most)) * inv
    return {"q": torch.round(t * per[:, None]).to(torch.int8), "scales": scales, "residual": stored}


def _act(v, name):
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v * (1.0 / (1.0 + torch.exp(-v))) if name == "silu" else v


def _mx(s):
    cin = s.case["cin"]
    values, exponent = _quantize(s.x)
    x = torch.ldexp(values, exponent[:, :, None]).flatten(1)[:, :cin].contiguous()
    return _act(x @ _unpack(s.w, s.w_scales, cin).t() + s.bias, s.case["act"]).to(s.x.dtype)


def _mxq(s):
    codes, scales = _pack(*_quantize(s.x))
    return _unpack(codes, scales, s.case["cin"]).to(s.x.dtype)


def _ancestors(parents):
    """[sequences, tokens, tokens]: whether the second token is the first or above it in the tree."""
    tokens = parents.shape[1]
    at = torch.arange(tokens, device=parents.device)
    near = ((at[None, None, :] == at[None, :, None]) | (at[None, None, :] == parents[:, :, None])).float()
    for _ in range(max(tokens - 1, 1).bit_length()):  # paths twice as long each time
        near = ((near @ near) > 0).float()
    return near > 0


def _tree(s):
    c = s.case
    heads, kv, d = c["heads"], c["kv_heads"], c["head_dim"]
    group = heads // kv
    q_len, k_len = s.cu_q[1:] - s.cu_q[:-1], s.cache_len
    items, tokens, cached = q_len.numel(), max(_ints(c["q"])), max(_ints(c["k"]))
    # Padded: [sequence, token] and [sequence, cached key, then token].
    t, j = torch.arange(tokens, device="cuda"), torch.arange(cached, device="cuda")
    row = (s.cu_q[:-1, None] + t).clamp_max(s.q.shape[0] - 1)
    key = (s.cache_start[:, None] + j).clamp_max(s.k_cache.shape[0] - 1)
    q = s.q[row].float().reshape(items, tokens, kv, group, d).permute(0, 2, 3, 1, 4).reshape(items * kv, group * tokens, d)
    k = torch.cat([s.k_cache[key], s.k[row]], 1).float().reshape(items, -1, kv, d).permute(0, 2, 3, 1).reshape(items * kv, d, -1)
    score = (torch.bmm(q.contiguous(), k.contiguous()) * s.scale).reshape(items, heads, tokens, -1)
    if c["cap"] > 0.0:
        score = c["cap"] * torch.tanh(score / c["cap"])
    if c["bias"]:
        at = s.positions[row]
        away = at[:, :, None] - torch.cat([j.expand(items, -1), at], 1)[:, None, :]
        score = score - s.slopes[None, :, None, None] * away.abs().float()[:, None]
    live = t[None, :] < q_len[:, None]
    parents = torch.where(live, s.parents[row], torch.full_like(row, -1, dtype=torch.int32))
    seen = torch.cat([(j < k_len[:, None])[:, None, :].expand(-1, tokens, -1), _ancestors(parents)], 2)
    score = score.masked_fill(~seen[:, None], -math.inf)
    p = torch.exp(score - score.amax(3, keepdim=True))
    p = (p / p.sum(3, keepdim=True)).reshape(items * kv, group * tokens, -1)
    v = torch.cat([s.v_cache[key], s.v[row]], 1).float()
    v = torch.where(torch.cat([j < k_len[:, None], live], 1)[:, :, None], v, torch.zeros_like(v))  # rows of others
    v = v.reshape(items, -1, kv, d).permute(0, 2, 1, 3).reshape(items * kv, -1, d)
    o = torch.bmm(p, v.contiguous()).reshape(items, heads, tokens, d).permute(0, 2, 1, 3)
    return o.reshape(items, tokens, heads * d)[live].to(s.q.dtype)


# ---- what a call cannot do without ------------------------------------------------

def work(case):
    if case["kind"] == "norm":
        values = case["rows"] * case["channels"]
        stream = 2 * SIZE[case["residual"]] if case["residual"] != "none" else 0
        out = 1 if case["out"] == "i8" else SIZE[case["x"]]
        # x, the residual in and out, the rows out and their scales, the gains.
        return {"bytes": values * (SIZE[case["x"]] + stream + out) + 4 * case["rows"] * (case["out"] == "i8") +
                4 * case["channels"], "flops": 5 * values}
    if case["kind"] == "mx":
        size, rows, cin, cout = SIZE[case["dtype"]], case["rows"], case["cin"], case["cout"]
        blocks = (cin + 31) // 32
        # x in, weights with scales and bias in, y out.
        return {"bytes": rows * cin * size + cout * (17 * blocks + 4) + rows * cout * size, "flops": 2 * rows * cin * cout}
    if case["kind"] == "mxq":
        values, blocks = case["rows"] * case["cin"], case["rows"] * ((case["cin"] + 31) // 32)
        # Values in and out; codes and scales written.
        return {"bytes": 2 * values * SIZE[case["dtype"]] + 17 * blocks, "flops": 4 * values}
    q_len, k_len = _ints(case["q"]), _ints(case["k"])
    heads, kv, d, size = case["heads"], case["kv_heads"], case["head_dim"], SIZE[case["dtype"]]
    # q in and o out, the tokens' and the caches' keys and values in, parents in.
    pairs = sum(n * (m + 1) for n, m in zip(q_len, k_len))  # (a token has at least itself of the tree)
    return {"bytes": 2 * (sum(q_len) * heads + (sum(q_len) + sum(k_len)) * kv) * d * size + 4 * sum(q_len),
            "flops": 4 * d * pairs * heads}


# ---- the same in 64 bits -------------------------------------------------------------

def _exact_blocks(x):
    """The values that the 4-bit blocks of x stand for, from the definition: the nearest of the eight
    magnitudes, of two as near that with the even code."""
    rows, channels = x.shape
    blocks = (channels + 31) // 32
    wide = torch.zeros((rows, blocks * 32), dtype=torch.float64, device=x.device)
    wide[:, :channels] = x.double()
    wide = wide.view(rows, blocks, 32)
    most = wide.abs().max(dim=2, keepdim=True).values
    scale = torch.exp2((torch.frexp(most).exponent - 1).double() - 2.0).clamp_min(2.0 ** -127)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    half = (grid[1:] + grid[:-1]) / 2.0
    size = wide.abs() / scale
    low, high = torch.bucketize(size, half, right=False), torch.bucketize(size, half, right=True)
    code = torch.where(low == high, low, torch.where(low % 2 == 0, low, high))
    return (grid[code] * scale * torch.sign(wide)).view(rows, blocks * 32)[:, :channels]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h, stored = s.x.double(), None
        if s.residual is not None:
            stored = h + s.residual.double()
            h = stored.to(s.residual.dtype).double()  # the norm is that of the stored rows
        length = torch.sqrt(h.square().sum(1) / case["channels"] + EPS)
        y = h * s.gamma.double() / length[:, None]
        if case["out"] == "y":
            return {"y": y, "residual": stored}
        # (The 8-bit values are defined by 32-bit arithmetic.)
        most = (h * s.gamma.double()).abs().max(dim=1).values
        return {"q": None, "scales": torch.where(most < 2.0 ** -100, 0.0, most / length / 127.0), "residual": stored}
    if case["kind"] == "mxq":
        return _exact_blocks(s.x)
    if case["kind"] == "mx":
        cin = case["cin"]
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
        grid = torch.cat([grid, -grid])
        w = torch.empty((case["cout"], s.w.shape[1] * 2), dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = grid[(s.w % 16).long()], grid[(s.w // 16).long()]
        w *= torch.exp2(s.w_scales.double() - 127.0).repeat_interleave(32, dim=1)[:, :w.shape[1]]
        w = w[:, :cin].contiguous()
        v = torch.empty((case["rows"], case["cout"]), dtype=torch.float64, device="cuda")
        for r0 in range(0, case["rows"], 8192):
            v[r0:r0 + 8192] = torch.nn.functional.linear(_exact_blocks(s.x[r0:r0 + 8192]), w, s.bias.double())
        if case["act"] == "gelu":
            v = v / (1.0 + torch.exp(-math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3)))
        elif case["act"] == "silu":
            v = v / (1.0 + torch.exp(-v))
        return v
    q_len, k_len = _ints(case["q"]), _ints(case["k"])
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros((sum(q_len), heads, d), dtype=torch.float64, device="cuda")
    parents = s.parents.tolist()
    for first, n, at, m in zip(_starts(q_len), q_len, s.cache_start.tolist(), k_len):
        hidden = torch.ones((n, m + n), dtype=torch.bool)
        hidden[:, :m] = False
        for i in range(n):
            j = i
            while j >= 0:
                hidden[i, m + j] = False
                j = parents[first + j]
        hidden = hidden.cuda()
        where = torch.cat([torch.arange(m, device="cuda"), s.positions[first:first + n]]).double()
        for h in range(heads):
            col = slice((h // (heads // kv)) * d, (h // (heads // kv) + 1) * d)
            k = torch.cat([s.k_cache[at:at + m, col], s.k[first:first + n, col]]).double()
            v = torch.cat([s.v_cache[at:at + m, col], s.v[first:first + n, col]]).double()
            z = torch.mm(s.q[first:first + n, h * d:(h + 1) * d].double(), k.t().contiguous()) * s.scale
            if case["cap"] > 0.0:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if case["bias"]:
                z = z - (where[None, :] - where[m:, None]).abs() * float(s.slopes[h])
            out[first:first + n, h] = torch.mm(torch.softmax(z.masked_fill(hidden, -math.inf), dim=1), v)
    return out.flatten(1)
