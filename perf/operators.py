"""The operators around the quantized linears of a decode step: what is measured, and their plain forms.

Three operators, used one after the other in every layer of a decoder that serves many streams:

``norm``    h = x + residual; RMSNorm(h) * weight in 8 bits with one scale a row, ready for the e4m3 or
            int8 linears (``qtts_b200.quant.kernels.add_rms_norm_quant``);
``rope``    the fused projection's output [q | k | v]: RMSNorm of each q and k head, rotary positions with
            several axes, q handed on, k and v written to a paged cache in 4 bits
            (``qtts_b200.kv4.rope_kv4_append``);
``attend``  attention of one or many new tokens over that cache (``qtts_b200.kv4.kv4_attention``).

The 4-bit cache. Keys and values are held apart, each as codes [pages, kv_heads, page_size, head_dim / 2]
(uint8, two codes a byte) and params [pages, kv_heads, page_size, head_dim / 32, 2] (bf16: scale, minimum).
32 neighbouring channels of one token and head share a scale and a minimum: value = code * scale + minimum,
code in 0..15. With j = channel // 32 and n = head_dim // 32, a key's channel 32j + 8c + i is nibble i (from
the low end) of 32-bit word c * n + j of its row; a value's channel 32j + 4g + i is nibble i of 16-bit word
g * n + j.
"""

from __future__ import annotations

import math
import sys

import torch

own = False

GROUP = 32  # channels that share a scale and a minimum
BASE = 1.0e6  # rotary base
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases ------------------------------------------------------------------------------------


def _attend(name, batch, lo, hi, q_len, heads, kv_heads, head_dim, page, dtype, causal=True):
    return {"name": name, "op": "attend", "batch": batch, "len_lo": lo, "len_hi": hi, "q_len": q_len, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "causal": causal}


def _rope(name, tokens, heads, kv_heads, head_dim, axes, interleaved, page, dtype):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "axes": axes, "interleaved": interleaved, "page": page, "dtype": dtype}


def _norm(name, rows, width, to, dtype):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "to": to, "dtype": dtype}


def listed():
    return [
        # One stream that has just begun: a call's latency is all that counts.
        _attend("attend one short stream", 1, 33, 33, 1, 16, 8, 128, 16, "bf16"),
        # The decode step of the frame benchmark: 8 streams, 512 earlier tokens, a slot cache of 768.
        _attend("attend slot cache", 8, 513, 513, 1, 16, 8, 128, 768, "bf16"),
        # A busy server: many streams of unlike lengths.
        _attend("attend many ragged streams", 64, 17, 8192, 1, 16, 8, 128, 64, "bf16"),
        # Few streams with a very long past: the work has to be split along the cache.
        _attend("attend long past", 2, 131071, 131071, 1, 32, 8, 128, 256, "bf16"),
        # Prompts read at once, each token sees those before it.
        _attend("attend prompts", 4, 2048, 2048, 2048, 16, 8, 128, 64, "bf16"),
        # A ragged chunk of new tokens over an earlier part; smaller heads, wide sharing, the other type.
        _attend("attend chunk", 3, 1500, 5001, 193, 32, 4, 64, 48, "fp16"),
        # One new token.
        _rope("rope one token", 1, 16, 8, 128, 1, False, 16, "bf16"),
        # Prompts with three axes in sections.
        _rope("rope prompts", 8192, 16, 8, 128, 3, False, 64, "bf16"),
        # A batch of new tokens, interleaved axes, smaller heads, the other type.
        _rope("rope small heads", 333, 32, 4, 64, 3, True, 48, "fp16"),
        # The hidden row of one stream, before an e4m3 linear.
        _norm("norm one row", 1, 2048, "e4m3", "bf16"),
        # Prompts, before an e4m3 linear.
        _norm("norm prompts", 16384, 2048, "e4m3", "bf16"),
        # A chunk of a wide model, before an int8 linear.
        _norm("norm wide int8", 777, 6144, "int8", "fp16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "rope", "norm"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm":
        width = rng.choice([8 * _log_int(rng, 64, 1024), _log_int(rng, 512, 8192)])
        rows = _log_int(rng, 1, (16384 * 2048) // width)
        case = _norm("", rows, width, rng.choice(["e4m3", "e4m3", "int8"]), dtype)
    else:
        head_dim = rng.choice([64, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 2, 4, 5, 8])
        page = rng.choice([16, 48, 64, 128, 256])
        if op == "rope":
            tokens = _log_int(rng, 1, min(8192, (8192 * 32 * 128) // ((heads + 2 * kv_heads) * head_dim)))
            axes = rng.choice([1, 3])
            case = _rope("", tokens, heads, kv_heads, head_dim, axes, axes == 3 and rng.random() < 0.5, page, dtype)
        elif rng.random() < 0.6:  # single tokens
            batch = _log_int(rng, 1, 128)
            hi = _log_int(rng, 1, min(131071, (262142 * 8) // (kv_heads * batch)))
            case = _attend("", batch, rng.choice([hi, max(1, hi // 20)]), hi, 1, heads, kv_heads, head_dim, page, dtype)
        else:  # several new tokens a stream
            batch = _log_int(rng, 1, 6)
            q_len = _log_int(rng, 2, 2048)
            most = (4 * 2048 * 2048 * 6) // (batch * q_len * heads)
            hi = max(q_len, _log_int(rng, 8, max(9, min(16384, most))))
            q_len = max(2, min(q_len, most))
            case = _attend("", batch, max(q_len, hi // 3), max(q_len, hi), q_len, heads, kv_heads, head_dim, page, dtype,
                           rng.random() < 0.8)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _quantize4(x):
    """x [..., D] fp32 -> codes [..., D] (whole numbers in fp32), scale and minimum [..., D / 32] bf16."""
    xg = x.unflatten(-1, (-1, GROUP))
    lo, hi = xg.amin(-1), xg.amax(-1)
    scale = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16)  # a division, not a product with 1/15
    low = lo.to(torch.bfloat16)
    s = scale.float()[..., None]
    codes = torch.clamp(torch.round((xg - low.float()[..., None]) / torch.where(s > 0, s, torch.ones_like(s))), 0, 15)
    return codes.flatten(-2), scale, low


def _pack(codes, keys):
    """codes [..., D] -> uint8 [..., D / 2] in the cache's order (see the top)."""
    n = codes.shape[-1] // GROUP
    run = 8 if keys else 4  # channels that stay together in one word
    c = codes.to(torch.uint8).unflatten(-1, (n, GROUP // run, run)).transpose(-3, -2).flatten(-3)
    c = c.unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


def _unpack(packed, keys):
    """The other way: uint8 [..., D / 2] -> codes [..., D] fp32."""
    n = packed.shape[-1] * 2 // GROUP
    run = 8 if keys else 4
    c = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    return c.unflatten(-1, (GROUP // run, n, run)).transpose(-3, -2).flatten(-3).float()


def _values(codes, params, keys):
    p = params.float()
    c = _unpack(codes, keys).unflatten(-1, (-1, GROUP))
    return (c * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _lengths(case):
    """One length a stream, spread over [len_lo, len_hi] (its logarithm), the longest among them."""
    b, lo, hi = case["batch"], case["len_lo"], case["len_hi"]
    return [int(round(lo * (hi / lo) ** (i / max(1, b - 1)))) if b > 1 else hi for i in range(b)]


def _q_lens(case):
    """New tokens a stream: all of q_len, or q_len and fewer where several streams bring a chunk."""
    b, q = case["batch"], case["q_len"]
    return [q if q % 2 == 0 or q == 1 else max(1, q - 37 * i) for i in range(b)]


def prepare(case, seed):
    g = _gen(seed)
    dev = "cuda"

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if case["op"] == "norm":
        dtype = DTYPES[case["dtype"]]
        rows, width = case["rows"], case["width"]
        return {"op": "norm", "to": case["to"], "x": (0.5 * randn(rows, width)).to(dtype),
                "residual": (2.0 * randn(rows, width)).to(dtype), "weight": (1.0 + 0.2 * randn(width)).to(dtype)}

    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    state = {"op": case["op"], "heads": heads, "kv_heads": kv_heads, "head_dim": d}
    if case["op"] == "rope":
        t = case["tokens"]
        pages = -(-t // page) + 2
        where = torch.randperm(pages * page, generator=g, device=dev)[:t]
        if t > 1:  # tokens of one page follow each other, as a prompt's do
            where = where.sort().values
        first = torch.randint(0, 1000, (case["axes"], 1), generator=g, device=dev)
        step = torch.arange(t, device=dev)[None, :].expand(case["axes"], t).clone()
        if case["axes"] > 1:  # height and width turn faster than time
            step[1] = step[1] // 7 % 61
            step[2] = step[2] % 7
        angles = torch.arange(16384, device=dev, dtype=torch.float32)[:, None] / BASE ** (
            torch.arange(0, d, 2, device=dev, dtype=torch.float32) / d)
        half = d // 2
        third = half // 4
        state.update(
            qkv=randn(t, (heads + 2 * kv_heads) * d).to(dtype), cos=torch.cos(angles), sin=torch.sin(angles),
            positions=first + step, slots=where, interleaved=case["interleaved"],
            sections=(half,) if case["axes"] == 1 else (half - 2 * third, third, third),
            q_norm=(1.0 + 0.2 * randn(d)).to(dtype), k_norm=(1.0 + 0.2 * randn(d)).to(dtype))
        for name in ("k", "v"):
            state[name + "_codes"] = torch.zeros(pages, kv_heads, page, d // 2, dtype=torch.uint8, device=dev)
            state[name + "_params"] = torch.zeros(pages, kv_heads, page, d // GROUP, 2, dtype=torch.bfloat16, device=dev)
        return state

    lengths, q_lens = _lengths(case), _q_lens(case)
    per = -(-max(lengths) // page)
    used = sum(-(-n // page) for n in lengths)
    order = torch.randperm(used, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(case["batch"], per, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(lengths):
        m = -(-n // page)
        table[i, :m] = order[at : at + m]
        at += m
    # Keys with a few strong channels, as trained models have them.
    loud = 1.0 + 3.0 * (torch.rand(kv_heads, 1, d, generator=g, device=dev) > 0.95)
    for name in ("k", "v"):
        codes = torch.empty(used, kv_heads, page, d // 2, dtype=torch.uint8, device=dev)
        params = torch.empty(used, kv_heads, page, d // GROUP, 2, dtype=torch.bfloat16, device=dev)
        step = max(1, (1 << 26) // (kv_heads * page * d))
        for i in range(0, used, step):
            x = randn(min(step, used - i), kv_heads, page, d) * (loud if name == "k" else 1.0)
            c, s, low = _quantize4(x)
            codes[i : i + step] = _pack(c, name == "k")
            params[i : i + step] = torch.stack((s, low), -1)
        state[name + "_codes"], state[name + "_params"] = codes, params
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    state.update(
        q=randn(starts[-1], heads, d).to(dtype), table=table, causal=case["causal"], max_q=max(q_lens),
        lengths=torch.tensor(lengths, dtype=torch.int32, device=dev),
        q_starts=torch.tensor(starts, dtype=torch.int32, device=dev) if max(q_lens) > 1 else None)
    return state


# ---- one pass ---------------------------------------------------------------------------------

_framework = None


def _own():
    global _framework
    if _framework is None:
        if "tts-inference_b200" not in sys.path:
            sys.path.insert(0, "tts-inference_b200")
        from qtts_b200 import kv4
        from qtts_b200.quant import kernels

        _framework = (kv4, kernels)
    return _framework


def run(state):
    return {"norm": _run_norm, "rope": _run_rope, "attend": _run_attend}[state["op"]](state)


def _run_norm(s):
    if own:
        to = torch.int8 if s["to"] == "int8" else torch.float8_e4m3fn
        q, scale, h = _own()[1].add_rms_norm_quant(s["x"], s["residual"], s["weight"], 1e-6, dtype=to)
        if s["to"] == "int8":  # the values that the codes stand for
            q = torch.mul(q, scale, out=torch.empty_like(h))
        return {"q": q, "scale": scale, "residual": h}
    h = s["x"].float() + s["residual"].float()
    y = s["weight"].float() * (h * (1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)))
    most = 127.0 if s["to"] == "int8" else 448.0
    scale = y.abs().amax(-1, keepdim=True).clamp_min(1e-6) * (1.0 / most)
    q = y / scale
    if s["to"] == "int8":
        q = (torch.clamp(torch.round(q), -127, 127) * scale).to(s["x"].dtype)
    else:
        q = q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale, "residual": h.to(s["x"].dtype)}


def _axis_of(pairs, sections, interleaved, device):
    """The axis whose position turns each pair of channels."""
    j = torch.arange(pairs, device=device)
    if interleaved:  # t h w t h w ..., and time where height and width have had their share
        n = len(sections)
        share = torch.tensor(sections, device=device)[j % n] * n
        return torch.where(j < share, j % n, torch.zeros_like(j))
    return torch.bucketize(j, torch.tensor(sections, device=device).cumsum(0), right=True)


def _rms(x, weight, eps=1e-6):
    return weight.float() * (x * (1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)))


def _run_rope(s):
    if own:
        kv4 = _own()[0]
        cache = kv4.Kv4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])
        q, k, v = kv4.rope_kv4_append(
            s["qkv"], cache, s["slots"], s["heads"], cos=s["cos"], sin=s["sin"], positions=s["positions"],
            sections=s["sections"], interleaved=s["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
            values=True)
        return {"q": q, "k": k, "v": v, "k_params": s["k_params"], "v_params": s["v_params"]}
    d, heads, kv_heads = s["head_dim"], s["heads"], s["kv_heads"]
    x = s["qkv"].float().unflatten(-1, (-1, d))
    q, k, v = x.split([heads, kv_heads, kv_heads], dim=1)
    axis = _axis_of(d // 2, s["sections"], s["interleaved"], x.device)
    at = s["positions"][axis].t()  # [tokens, pairs]
    pair = torch.arange(d // 2, device=x.device)
    c, n = s["cos"][at, pair][:, None], s["sin"][at, pair][:, None]

    def turn(y):
        a, b = y.chunk(2, -1)
        return torch.cat((a * c - b * n, b * c + a * n), -1)

    q, k = turn(_rms(q, s["q_norm"])), turn(_rms(k, s["k_norm"]))
    page = s["k_codes"].shape[2]
    which, row = s["slots"] // page, s["slots"] % page
    held = {}
    for name, y in (("k", k), ("v", v)):
        codes, scale, low = _quantize4(y)
        s[name + "_codes"][which, :, row] = _pack(codes, name == "k")
        s[name + "_params"][which, :, row] = torch.stack((scale, low), -1)
        held[name] = (codes.unflatten(-1, (-1, GROUP)) * scale.float()[..., None] + low.float()[..., None]).flatten(-2)
    dtype = s["qkv"].dtype
    return {"q": q.to(dtype), "k": held["k"].to(dtype), "v": held["v"].to(dtype),
            "k_params": s["k_params"], "v_params": s["v_params"]}


def _run_attend(s):
    if own:
        kv4 = _own()[0]
        cache = kv4.Kv4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])
        return kv4.kv4_attention(s["q"], cache, s["table"], s["lengths"], q_starts=s["q_starts"], max_q=s["max_q"],
                                 causal=s["causal"])
    q, table, lengths = s["q"].float(), s["table"], s["lengths"].long()
    dev, heads, kv_heads, d = q.device, s["heads"], s["kv_heads"], s["head_dim"]
    page, batch = s["k_codes"].shape[2], table.shape[0]
    # Every stream padded to the longest past and to the most new tokens.
    most = table.shape[1] * page
    k = _values(s["k_codes"][table], s["k_params"][table], True).transpose(1, 2).reshape(batch, kv_heads, most, d)
    v = _values(s["v_codes"][table], s["v_params"][table], False).transpose(1, 2).reshape(batch, kv_heads, most, d)
    n = s["max_q"]
    starts = s["q_starts"].long() if s["q_starts"] is not None else torch.arange(batch + 1, device=dev)
    new = starts[1:] - starts[:-1]
    i = torch.arange(n, device=dev)
    there = i[None, :] < new[:, None]  # [batch, n]
    qp = q[torch.where(there, starts[:-1, None] + i, torch.zeros_like(starts[:-1, None]))]
    qp = qp.unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, d)
    score = (qp @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    score = score.view(batch, kv_heads, heads // kv_heads, n, most)
    sees = (lengths - new)[:, None] + i + 1 if s["causal"] else lengths[:, None].expand(batch, n)
    seen = torch.arange(most, device=dev) < sees[..., None]  # [batch, n, most]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    e = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    out = (e.view(batch, kv_heads, -1, most) @ v).view(batch, heads, n, d).transpose(1, 2)
    return out[there].to(s["q"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        # x and the residual read, the residual and the codes written, a scale a row, the weight once.
        return {"bytes": n * (2 + 2 + 2 + 1) + 4 * case["rows"] + 2 * case["width"], "flops": 8 * n}
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    row = d // 2 + 4 * (d // GROUP)  # a key or value of one head: its codes, scales and minima
    if case["op"] == "rope":
        t = case["tokens"]
        # The projection read; q, the cache's rows and the values that they stand for written.
        moved = 2 * (heads + 2 * kv_heads) * d + 2 * heads * d + 2 * kv_heads * (row + 2 * d) + 8 * (case["axes"] + 1)
        angles = 4 * d * (min(t, 16384) if case["axes"] == 1 else 1)
        return {"bytes": t * moved + angles, "flops": 10 * t * (heads + 2 * kv_heads) * d}
    lengths, q_lens = _lengths(case), _q_lens(case)
    pairs = 0
    for n, q in zip(lengths, q_lens):
        pairs += q * n - (q * (q - 1) // 2 if case["causal"] else 0)
    return {"bytes": 2 * kv_heads * row * sum(lengths) + 4 * heads * d * sum(q_lens), "flops": 4 * d * heads * pairs}


# ---- the same in 64 bits ------------------------------------------------------------------------


def _exact4(x):
    """x [..., D] in 64 bits -> the values that its 4-bit codes stand for, scale and minimum (bf16, as held)."""
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    least, most = blocks.min(-1).values, blocks.max(-1).values
    scale = ((most - least) / 15).to(torch.bfloat16)
    least = least.to(torch.bfloat16)
    s, z = scale.double().unsqueeze(-1), least.double().unsqueeze(-1)
    code = ((blocks - z) / torch.where(s > 0, s, torch.ones_like(s))).round().clamp(0, 15)
    return (code * s + z).reshape(x.shape), scale, least


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + s["residual"].double()
        y = h / (h.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * s["weight"].double()
        most = 127 if case["to"] == "int8" else 448
        scale = y.abs().max(1, keepdim=True).values.clamp_min(1e-6) / most
        if case["to"] == "int8":
            q = (y / scale).round().clamp(-127, 127) * scale
        else:
            q = (y / scale).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
        return {"q": q, "scale": scale, "residual": h}
    d, heads, kv_heads = case["head_dim"], case["heads"], case["kv_heads"]
    if case["op"] == "rope":
        t = case["tokens"]
        x = s["qkv"].double().view(t, heads + 2 * kv_heads, d)
        cos, sin = s["cos"].double(), s["sin"].double()
        turned = []
        for part, weight in ((x[:, :heads], s["q_norm"]), (x[:, heads : heads + kv_heads], s["k_norm"])):
            y = part / (part.pow(2).mean(2, keepdim=True) + 1e-6).sqrt() * weight.double()
            z = torch.empty_like(y)
            for j in range(d // 2):
                axis, left = 0, j
                if case["axes"] > 1 and case["interleaved"]:
                    axis = j % 3 if j < 3 * s["sections"][j % 3] else 0
                elif case["axes"] > 1:
                    while left >= s["sections"][axis]:
                        left -= s["sections"][axis]
                        axis += 1
                c, n = (f[s["positions"][axis], j].unsqueeze(1) for f in (cos, sin))
                a, b = y[:, :, j], y[:, :, j + d // 2]
                z[:, :, j], z[:, :, j + d // 2] = a * c - b * n, b * c + a * n
            turned.append(z)
        page = case["page"]
        out = {"q": turned[0]}
        for name, y in (("k", turned[1]), ("v", x[:, heads + kv_heads :])):
            held, scale, least = _exact4(y)
            params = s[name + "_params"].double()
            for part, what in ((0, scale), (1, least)):
                params[s["slots"] // page, :, s["slots"] % page, :, part] = what.double()
            out[name], out[name + "_params"] = held, params
        return out
    lengths, q_lens = _lengths(case), _q_lens(case)
    page, n, dev = case["page"], d // GROUP, "cuda"
    ch = torch.arange(d, device=dev)
    nibble = {"k": ((ch % 32 // 8) * n + ch // 32) * 8 + ch % 8, "v": ((ch % 32 // 4) * n + ch // 32) * 4 + ch % 4}
    out, at = [], 0
    for b in range(case["batch"]):
        pages = s["table"][b, : -(-lengths[b] // page)].long()
        kv = {}
        for name in ("k", "v"):
            byte = s[name + "_codes"][pages][..., nibble[name] // 2].int()
            code = (byte >> (4 * (nibble[name] % 2)).int()) & 15
            p = s[name + "_params"][pages].double()
            val = code.double() * p[..., ch // 32, 0] + p[..., ch // 32, 1]
            kv[name] = val.permute(1, 0, 2, 3).reshape(kv_heads, -1, d)[:, : lengths[b]]
        q = s["q"][at : at + q_lens[b]].double()
        at += q_lens[b]
        parts = []
        for h in range(heads):
            score = q[:, h] @ kv["k"][h * kv_heads // heads].T / math.sqrt(d)
            if case["causal"]:
                late = torch.ones(score.shape, dtype=torch.bool, device=dev).triu(lengths[b] - q_lens[b] + 1)
                score[late] = -math.inf
            parts.append(torch.softmax(score, 1) @ kv["v"][h * kv_heads // heads])
        out.append(torch.stack(parts, 1))
    return torch.cat(out)
