"""The parts of a transformer's attention layer over token sequences, served in
8 bits: what they are measured on.

Three kinds of case:
  linear  activations quantized row by row to 8-bit integers, then the product
          with 8-bit weights (a scale per token and per channel), bias and
          activation;
  rope    rotary positions of q and k heads (interleaved or half layout, the
          whole head or part of it, frequencies stretched for long contexts);
  attn    varlen attention with shared key/value heads whose scores are capped,
          biased by distance, causal or prefix-masked, for prompts and for
          single new tokens over long caches.

`prepare` makes what a caller holds before the call, `run` is one call (in
plain torch, or through the Python binding where `own` is set), `work` the
bytes and operations the call cannot do without, `exact` its outputs in 64
bits.  Widths, head counts and lengths are those of the flow model's blocks
(width 1024, MLP 4096, 16 heads of 64, 1,370 context tokens, up to 42k rows) or
generic.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
ACTS = {"none": 0, "gelu": 1, "silu": 2}


# ---- cases -----------------------------------------------------------------

def listed():
    return [
        # One new token through the first MLP linear of a block.
        dict(name="linear_token", kind="linear", dtype="bf16", rows=1, cin=1024, cout=4096, act="gelu"),
        # A small object's tokens (or an image's 1,370) through the same linear.
        dict(name="linear_mlp_1370", kind="linear", dtype="bf16", rows=1370, cin=1024, cout=4096, act="gelu"),
        # The second MLP linear at the flow model's largest voxel count.
        dict(name="linear_42k", kind="linear", dtype="bf16", rows=42017, cin=4096, cout=1024, act="none"),
        # Odd sizes throughout, fp32 in and out: rows are no whole 16-byte pieces.
        dict(name="linear_odd_f32", kind="linear", dtype="f32", rows=4739, cin=1370, cout=1021, act="silu"),
        # A batch of single tokens at far positions of a stretched context.
        dict(name="rope_tokens", kind="rope", dtype="bf16", rows=16, heads=20, head_dim=128, rotary=128,
             layout="half", factor=8.0, far=131072),
        # q and k of a packed [rows, 3 C] projection of long sequences.
        dict(name="rope_32k", kind="rope", dtype="bf16", rows=32768, heads=32, head_dim=64, rotary=64,
             layout="interleaved", factor=1.0, far=20480),
        # Part of each head turned, odd row count, fp32.
        dict(name="rope_part_f32", kind="rope", dtype="f32", rows=9473, heads=16, head_dim=80, rotary=48,
             layout="half", factor=4.0, far=40000),
        # Prompts of a causal model with capped scores and shared key/value heads.
        dict(name="attn_prompt_cap", kind="attn", dtype="bf16", q="8192,2903,4739", k="8192,2903,4739", heads=16,
             kv_heads=4, head_dim=128, cap=30.0, bias=0, causal=1, prefix=""),
        # Image tokens seen by all, then causal tokens, with a bias by distance.
        dict(name="attn_prefix_bias", kind="attn", dtype="bf16", q="5466,3097", k="5466,3097", heads=16,
             kv_heads=16, head_dim=64, cap=0.0, bias=1, causal=1, prefix="1370,1370"),
        # One new token for each of a batch of ragged caches.
        dict(name="attn_tokens_long", kind="attn", dtype="bf16", q="1,1,1,1,1,1,1,1",
             k="65536,40001,32768,20480,9999,1370,17,1", heads=32, kv_heads=8, head_dim=128, cap=50.0, bias=0,
             causal=1, prefix=""),
        # One new token of one short sequence, every head its own keys.
        dict(name="attn_token_one", kind="attn", dtype="bf16", q="1", k="1501", heads=16, kv_heads=16, head_dim=64,
             cap=0.0, bias=1, causal=1, prefix=""),
        # fp32, a chunk of a prompt over its cache, everything at once.
        dict(name="attn_chunk_f32", kind="attn", dtype="f32", q="1000,517", k="2370,517", heads=16, kv_heads=8,
             head_dim=64, cap=20.0, bias=1, causal=1, prefix="1370,100"),
    ]


def draw(rng: random.Random):
    """One more case of the listed kinds, over the whole range of sizes."""

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["linear", "rope", "attn", "attn"])
    if kind == "linear":
        cin = rng.choice([rng.randint(33, 500), 1024, 1370, rng.randint(500, 4096), 4096])
        cout = rng.choice([rng.randint(8, 300), 1024, 1021, rng.randint(300, 4096), 4096])
        most = 42017 * 4096 * 1024 // (cin * cout)
        return dict(kind=kind, dtype=rng.choice(["f32", "bf16", "bf16"]), rows=log(1, min(42017, max(most, 1))),
                    cin=cin, cout=cout, act=rng.choice(["none", "gelu", "silu"]))
    if kind == "rope":
        head_dim = rng.choice([64, 80, 96, 128, 128])
        rotary = rng.choice([head_dim, head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)])
        heads = rng.randint(1, 32)
        return dict(kind=kind, dtype=rng.choice(["f32", "bf16", "bf16"]),
                    rows=log(1, 32768 * 2048 // (heads * head_dim * 2)), heads=heads, head_dim=head_dim,
                    rotary=rotary, layout=rng.choice(["interleaved", "half"]),
                    factor=rng.choice([1.0, 2.0, 8.0, 32.0]), far=log(100, 1000000))
    dtype = rng.choice(["f32", "bf16", "bf16", "bf16"])
    head_dim = rng.choice([64, 64, 128, 128, 80, 96])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 3])
    items = rng.randint(1, 8)
    if rng.random() < 0.5:  # new tokens, a few at a time, over caches
        q = [rng.choice([1, 1, 1, 2, 5]) for _ in range(items)]
        k = [log(1, 40000) for _ in range(items)]
    else:
        top = 2000 if dtype == "f32" else 5000 if heads <= 8 else 3500
        q = [log(1, top) for _ in range(items)]
        k = [n + rng.choice([0, 0, rng.randint(0, 2000)]) for n in q]
    causal = rng.choice([0, 1, 1])
    prefix = ",".join(str(rng.randint(0, n)) for n in k) if causal and rng.random() < 0.4 else ""
    return dict(kind=kind, dtype=dtype, q=",".join(map(str, q)), k=",".join(map(str, k)), heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                bias=rng.choice([0, 1]), causal=causal, prefix=prefix)


def _ints(text):
    return [int(n) for n in text.split(",")] if text else []


# ---- inputs -----------------------------------------------------------------

class _State(dict):
    __getattr__ = dict.__getitem__


def _binding():
    folder = str(Path(__file__).resolve().parents[1] / "pixal3d.cpp_amd" / "python")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import pxs
    return pxs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    dtype = DTYPES[case["dtype"]]
    s = _State(case=case)
    if case["kind"] == "linear":
        rows, cin, cout = case["rows"], case["cin"], case["cout"]
        # Tokens of different size, a few channels an order larger than the rest.
        channel = torch.exp(0.5 * rand(cin))
        channel[torch.randint(0, cin, (max(cin // 128, 1),), device="cuda", generator=gen)] *= 10.0
        s.x = (rand(rows, cin) * channel * torch.exp(0.3 * rand(rows, 1))).to(dtype)
        # Weights quantized once, when the model was loaded.
        w = rand(cout, cin) * (torch.exp(0.3 * rand(cout, 1)) / math.sqrt(cin))
        s.w, s.w_scales = _quantize(w)
        s.bias = 0.1 * rand(cout)
        s.y = torch.empty((rows, cout), dtype=dtype, device="cuda")
        s.xq = torch.empty((rows, cin), dtype=torch.int8, device="cuda")
        s.x_scales = torch.empty(rows, dtype=torch.float32, device="cuda")
    elif case["kind"] == "rope":
        rows, width = case["rows"], case["heads"] * case["head_dim"]
        # q and k, then as much again as half of them for v, in one projection.
        s.qkv = rand(rows, width + width // 2 // 8 * 8).to(dtype)
        s.x = s.qkv[:, :width]
        start = torch.randint(0, case["far"], (rows // 512 + 1,), device="cuda", generator=gen)
        s.positions = (start.repeat_interleave(512)[:rows] + torch.arange(rows, device="cuda") % 512).to(torch.int32)
        s.freq = _frequencies(case["rotary"], 10000.0, case["factor"], 4096.0, 1.0, 32.0)
        s.magnitude = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
        s.y = torch.empty((rows, width), dtype=dtype, device="cuda")
    else:
        q_len, k_len = _ints(case["q"]), _ints(case["k"])
        heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        # Scores of a few units, as normalised q and k with learned gains give.
        s.q = (2.0 * rand(sum(q_len), heads * d)).to(dtype)
        s.kv = rand(sum(k_len), 2 * kv * d)
        s.kv[:, :kv * d] *= 2.0
        s.kv = s.kv.to(dtype)
        s.k, s.v = s.kv[:, :kv * d], s.kv[:, kv * d:]
        s.o = torch.empty((sum(q_len), heads * d), dtype=dtype, device="cuda")
        bounds = lambda n: torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int64, device="cuda")  # noqa: E731
        s.cu_q, s.cu_k = bounds(q_len), bounds(k_len)
        s.scale = 1.0 / math.sqrt(d)
        s.slopes = None
        if case["bias"]:
            s.slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)
        s.prefix = torch.tensor(_ints(case["prefix"]), dtype=torch.int64, device="cuda") if case["prefix"] else None
    if own:
        pxs = _binding()
        s.px = pxs.Pxs()
        if case["kind"] == "rope":
            s.layout = {"interleaved": pxs.ROPE_INTERLEAVED, "half": pxs.ROPE_HALF}[case["layout"]]
        if case["kind"] == "attn":
            s.workspace = s.px.attention_scores_workspace(len(q_len), sum(q_len), sum(k_len), heads, kv, d,
                                                          device="cuda")
    return s


def _quantize(x):
    """8-bit rows: largest magnitude to 127, ties to even -> (int8, fp32 scales)."""
    x = x.float()
    most = x.abs().amax(1, keepdim=True)
    live = most >= 2.0 ** -100
    # Divisions of tensors, each rounded once (by a number, torch multiplies with its inverse).
    top = torch.full_like(most, 127.0)
    per = torch.where(live, top / most.clamp_min(2.0 ** -100), torch.zeros_like(most))
    scales = torch.where(live, most / top, torch.zeros_like(most))
    return torch.round(x * per).to(torch.int8), scales[:, 0].contiguous()


def _frequencies(rotary, base, factor, length, low, high):
    """Angle per position of each pair: base^(-2 i / rotary); those that make few
    turns over the original length are slowed down by the factor."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64)
    freq = base ** (-i / rotary)
    if factor != 1.0:
        turns = length * freq / (2.0 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
    return freq.cuda()


# ---- one call ------------------------------------------------------------------

def run(s):
    kind = s.case["kind"]
    if own:
        return {"linear": _own_linear, "rope": _own_rope, "attn": _own_attn}[kind](s)
    return {"linear": _linear, "rope": _rope, "attn": _attn}[kind](s)


def _own_linear(s):
    s.px.quantize_rows(s.x, out=s.xq, scales=s.x_scales)
    s.px.linear_i8(s.xq, s.x_scales, s.w, s.w_scales, s.bias, ACTS[s.case["act"]], out=s.y)
    return {"y": s.y, "q": s.xq, "scales": s.x_scales}


def _own_rope(s):
    c = s.case
    return s.px.rope_positions(s.x, s.positions, s.freq, c["heads"], c["head_dim"], s.layout, s.magnitude, out=s.y)


def _own_attn(s):
    c = s.case
    return s.px.varlen_attention_scores(s.q, s.k, s.v, s.cu_q, s.cu_k, c["heads"], c["kv_heads"], c["head_dim"],
                                        s.scale, cap=c["cap"], slopes=s.slopes, causal=bool(c["causal"]),
                                        prefix=s.prefix, out=s.o, workspace=s.workspace)


def _act(v, name):
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v * (1.0 / (1.0 + torch.exp(-v))) if name == "silu" else v


def _linear(s):
    q, scales = _quantize(s.x)
    v = (q.float() @ s.w.float().t()) * scales[:, None] * s.w_scales[None, :] + s.bias
    return {"y": _act(v, s.case["act"]).to(s.x.dtype), "q": q, "scales": scales}


def _rope(s):
    c = s.case
    x = s.x.float().reshape(c["rows"], c["heads"], c["head_dim"])
    angle = s.positions.double()[:, None] * s.freq[None, :]
    cos = (torch.cos(angle) * s.magnitude).float()[:, None, :]
    sin = (torch.sin(angle) * s.magnitude).float()[:, None, :]
    y = x.clone()
    r = c["rotary"]
    a, b = (slice(0, r, 2), slice(1, r, 2)) if c["layout"] == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y.reshape(c["rows"], -1).to(s.x.dtype)


def _attn(s, wide=torch.float32):
    c = s.case
    heads, kv, d = c["heads"], c["kv_heads"], c["head_dim"]
    out = torch.empty((s.q.shape[0], heads * d), dtype=wide, device=s.q.device)
    q_len, k_len, prefix = _ints(c["q"]), _ints(c["k"]), _ints(c["prefix"])
    q0 = k0 = 0
    for i, (nq, nk) in enumerate(zip(q_len, k_len)):
        q = s.q[q0:q0 + nq].to(wide).reshape(nq, heads, d).transpose(0, 1)
        k = s.k[k0:k0 + nk].to(wide).reshape(nk, kv, d).transpose(0, 1)
        v = s.v[k0:k0 + nk].to(wide).reshape(nk, kv, d).transpose(0, 1).contiguous()
        pk = torch.arange(nk, device=q.device)
        for h in range(kv):
            g = heads // kv
            score = s.scale * (q[h * g:(h + 1) * g].reshape(g * nq, d) @ k[h].t().contiguous()).reshape(g, nq, nk)
            if c["cap"] > 0.0:
                score = c["cap"] * torch.tanh(score / c["cap"])
            pq = torch.arange(nk - nq, nk, device=q.device)
            if c["bias"]:
                away = (pq[:, None] - pk[None, :]).abs().to(wide)
                score = score - s.slopes[h * g:(h + 1) * g].to(wide)[:, None, None] * away
            if c["causal"]:
                seen = pk[None, :] <= pq[:, None]
                if prefix:
                    seen = seen | (pk[None, :] < prefix[i])
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
            top = score.amax(2, keepdim=True)
            p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = p.sum(2, keepdim=True)
            o = (p.reshape(g * nq, nk) @ v[h]).reshape(g, nq, d) / torch.where(total == 0.0, torch.ones_like(total), total)
            out[q0:q0 + nq].reshape(nq, heads, d)[:, h * g:(h + 1) * g] = o.transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    return out.to(s.q.dtype)


# ---- what a call cannot do without ------------------------------------------------

def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "linear":
        rows, cin, cout = case["rows"], case["cin"], case["cout"]
        # x in, its 8-bit form and scales out, weights, scales and bias in, y out.
        return {"bytes": rows * cin * (size + 1) + 4 * rows + cout * (cin + 8) + rows * cout * size,
                "flops": 2 * rows * cin * cout}
    if case["kind"] == "rope":
        elements = case["rows"] * case["heads"] * case["head_dim"]
        turned = case["rows"] * case["heads"] * case["rotary"]
        return {"bytes": 2 * elements * size + 4 * case["rows"] + 4 * case["rotary"], "flops": 3 * turned}
    q_len, k_len, prefix = _ints(case["q"]), _ints(case["k"]), _ints(case["prefix"])
    d, pairs = case["head_dim"], 0
    for i, (nq, nk) in enumerate(zip(q_len, k_len)):
        if not case["causal"]:
            pairs += nq * nk
            continue
        first = prefix[i] if prefix else 0
        pairs += sum(max(min(max(p + 1, 0), nk), min(first, nk)) for p in range(nk - nq, nk))
    return {"bytes": (2 * sum(q_len) * case["heads"] + 2 * sum(k_len) * case["kv_heads"]) * d * size,
            "flops": 4 * d * pairs * case["heads"]}


# ---- the same in 64 bits -------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        # The 8-bit values are defined by 32-bit arithmetic: one rounded division a
        # row, one rounded product an element (each rounded once from 64 bits here).
        x = s.x.double()
        most = x.abs().max(dim=1).values
        dead = most < 2.0 ** -100
        per = torch.where(dead, 0.0, (127.0 / most.masked_fill(dead, 1.0)).float().double())
        q = (x * per[:, None]).float().double().round()
        v = torch.empty((case["rows"], case["cout"]), dtype=torch.float64, device="cuda")
        w = s.w.double()
        for r0 in range(0, case["rows"], 8192):
            v[r0:r0 + 8192] = torch.nn.functional.linear(q[r0:r0 + 8192], w)
        v = v * torch.outer(torch.where(dead, 0.0, most / 127.0), s.w_scales.double()) + s.bias.double()
        if case["act"] == "gelu":
            v = v / (1.0 + torch.exp(-math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3)))
        elif case["act"] == "silu":
            v = v / (1.0 + torch.exp(-v))
        return {"y": v, "q": None, "scales": torch.where(dead, 0.0, most / 127.0)}
    if case["kind"] == "rope":
        r = case["rotary"]
        turn = torch.polar(torch.full_like(s.freq, s.magnitude).expand(case["rows"], -1).contiguous(),
                           torch.outer(s.positions.double(), s.freq))[:, None, :]
        y = s.x.double().reshape(case["rows"], case["heads"], case["head_dim"]).clone()
        head = y[..., :r]
        if case["layout"] == "half":
            z = torch.complex(head[..., :r // 2], head[..., r // 2:]) * turn
            y[..., :r] = torch.cat([z.real, z.imag], dim=-1)
        else:
            z = torch.view_as_complex(head.reshape(*head.shape[:2], r // 2, 2).contiguous()) * turn
            y[..., :r] = torch.view_as_real(z).flatten(2)
        return y.reshape(case["rows"], -1)
    q_len, k_len, prefix = _ints(case["q"]), _ints(case["k"]), _ints(case["prefix"])
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros((sum(q_len), heads, d), dtype=torch.float64, device="cuda")
    q_at = k_at = 0
    for i, (nq, nk) in enumerate(zip(q_len, k_len)):
        key = torch.arange(nk, dtype=torch.float64, device="cuda")
        for h in range(heads):
            k = s.k[k_at:k_at + nk, (h // (heads // kv)) * d:][:, :d].double()
            v = s.v[k_at:k_at + nk, (h // (heads // kv)) * d:][:, :d].double()
            for first in range(0, nq, 4096):
                rows = min(4096, nq - first)
                q = s.q[q_at + first:q_at + first + rows, h * d:(h + 1) * d].double()
                at = torch.arange(first, first + rows, dtype=torch.float64, device="cuda")[:, None] + (nk - nq)
                z = torch.mm(q, k.t().contiguous()) * s.scale
                if case["cap"] > 0.0:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                if case["bias"]:
                    z = z - (key - at).abs() * float(s.slopes[h])
                if case["causal"]:
                    hidden = key > at
                    if prefix:
                        hidden = hidden & (key >= prefix[i])
                    z = z.masked_fill(hidden, -math.inf)
                p = torch.softmax(z, dim=1).nan_to_num(0.0)
                out[q_at + first:q_at + first + rows, h] = torch.mm(p, v)
        q_at, k_at = q_at + nq, k_at + nk
    return out.flatten(1)
