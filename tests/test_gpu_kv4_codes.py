"""The codes that the cache writer stores, bit for bit.

The writer states its formula step by step, each step rounded once to fp32:
  inv = 1 / sqrt(mean(x^2) + eps);  y = w * (x * inv);  (a c - b s, b c + a s) of a pair;
  scale = bf16((max - min) / 15), minimum = bf16(min), code = clamp(rne((y - minimum) / scale), 0, 15)
and the sum of squares in one order (four neighbours at a time for 128 channels, then halves of
the row added to each other until one is left). The same steps as torch operations, one
kernel each, in fp32, have to give the same q, parameters and stored values: there is nothing left
to round differently, so the bar is equality.

A key is also held to 64 bits: away from the boundary between two codes the code is the exact
one. fp32 moves (y - minimum) / scale by some 6 roundings of values up to 15 steps: 15 * 6 * 2^-24
< 1e-5 steps, and a minimum or scale that rounds to another bf16 value is left out (the group's
parameters differ then, by one step of bf16 as both are within fp32's error of the boundary).
"""

from __future__ import annotations

import pytest
import torch

import kv4_reference as ref
from conftest import require_b200
from qtts_b200 import _native as nat
from qtts_b200 import kv4

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(autouse=True)
def _device():
    require_b200()
    nat.device_status(reset=True)
    yield
    torch.cuda.synchronize()
    assert nat.device_status(reset=True) == 0


def sum_of_squares(x):
    """[..., D] fp32 -> [..., 1], in the writer's order."""
    s = x * x
    if s.shape[-1] == 128:
        s = s.unflatten(-1, (32, 4))
        s = ((s[..., 0] + s[..., 1]) + s[..., 2]) + s[..., 3]
    while s.shape[-1] > 1:
        half = s.shape[-1] // 2
        s = s[..., :half] + s[..., half:]
    return s


def steps(x, weight, eps, cos, sin):
    """[T, H, D] in the activations' type -> fp32, one rounding a step; cos and sin [T, 1, D / 2]."""
    x = x.float()
    if weight is not None:
        inv = 1.0 / torch.sqrt(sum_of_squares(x) * (1.0 / x.shape[-1]) + eps)
        x = weight.float() * (x * inv)
    if cos is None:
        return x
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def quantized(x):
    """[..., D] fp32 -> the values stored, scale and minimum, in fp32 steps."""
    g = x.unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16)
    low = lo.to(torch.bfloat16)
    s, z = scale.float()[..., None], low.float()[..., None]
    code = torch.clamp(torch.round((g - z) / torch.where(s > 0, s, torch.ones_like(s))), 0, 15)
    return (code * s + z).flatten(-2), torch.stack((scale, low), -1), code


def inputs(tokens, heads, kv_heads, d, name, seed):
    g = torch.Generator().manual_seed(seed)
    dtype = DTYPES[name]
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * d, generator=g).to(dtype).cuda()
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(dtype).cuda() for _ in range(2))
    angle = torch.arange(4096, dtype=torch.float64)[:, None] / 1.0e6 ** (torch.arange(0, d, 2).double() / d)
    cos, sin = torch.cos(angle).float().cuda(), torch.sin(angle).float().cuda()
    at = torch.randint(0, 4096, (tokens,), generator=g).cuda()
    return qkv, qw, kw, cos, sin, at


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 16, 8), (333, 5, 3), (6000, 4, 8)])
@pytest.mark.parametrize("norm,rope", [(True, True), (True, False), (False, True)])
def test_codes_are_those_of_the_separate_steps(name, d, tokens, heads, kv_heads, norm, rope):
    qkv, qw, kw, cos, sin, at = inputs(tokens, heads, kv_heads, d, name, tokens + d)
    qw, kw = (qw, kw) if norm else (None, None)
    page = 64
    cache = kv4.Kv4Cache.empty(-(-tokens // page), kv_heads, page, d)
    slots = torch.arange(tokens).cuda()
    rope_args = dict(cos=cos, sin=sin, positions=at) if rope else {}
    q, k_held, v_held = kv4.rope_kv4_append(qkv, cache, slots, heads, q_norm=qw, k_norm=kw, eps=1e-6, values=True,
                                            **rope_args)
    c, s = (cos[at][:, None], sin[at][:, None]) if rope else (None, None)
    x = qkv.unflatten(1, (-1, d))
    assert torch.equal(q, steps(x[:, :heads], qw, 1e-6, c, s).to(q.dtype))
    keys = steps(x[:, heads : heads + kv_heads], kw, 1e-6, c, s)
    for want, held, params in ((keys, k_held, cache.k_params), (x[:, heads + kv_heads :].float(), v_held, cache.v_params)):
        value, pair, _ = quantized(want)
        assert torch.equal(params.transpose(1, 2).flatten(0, 1)[:tokens], pair)
        assert torch.equal(held, value.to(held.dtype))


@pytest.mark.parametrize("d", [64, 128])
def test_keys_have_the_codes_of_64_bits(d):
    tokens, kv_heads, page = 8192, 8, 64
    qkv, _, kw, cos, sin, at = inputs(tokens, 0, kv_heads, d, "bf16", 77)
    cache = kv4.Kv4Cache.empty(tokens // page, kv_heads, page, d)
    kv4.rope_kv4_append(qkv, cache, torch.arange(tokens).cuda(), 0, cos=cos, sin=sin, positions=at, k_norm=kw, eps=1e-6)
    x = qkv.unflatten(1, (-1, d))[:, :kv_heads].double()
    y = kw.double() * x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    a, b = y.chunk(2, -1)
    c, s = cos[at][:, None].double(), sin[at][:, None].double()
    y = torch.cat((a * c - b * s, b * c + a * s), -1)
    g = y.unflatten(-1, (-1, 32))
    params = cache.k_params.transpose(1, 2).flatten(0, 1)
    scale = ((g.amax(-1) - g.amin(-1)) / 15).to(torch.bfloat16)
    low = g.amin(-1).to(torch.bfloat16)
    same = (params[..., 0] == scale) & (params[..., 1] == low)
    # Parameters that differ are on a boundary of bf16: some 2^-24 * 8 / 2^-8 of the groups.
    assert same.double().mean() >= 1 - 4 * 8 * 2.0**-16
    step = scale.double()[..., None]
    place = (g - low.double()[..., None]) / step
    sure = ((place - place.floor() - 0.5).abs() > 1e-5) & same[..., None]
    got = ref.read_rows(cache.k_codes, cache.k_params, True).transpose(1, 2).flatten(0, 1).unflatten(-1, (-1, 32))
    code = ((got - low.double()[..., None]) / step).round()
    assert torch.equal(code[sure], place.round().clamp(0, 15)[sure])


def test_a_refused_token_gives_zeros_without_eps():
    # Its outputs are zeros whatever the norm would make of a row of zeros.
    d = 64
    qkv, qw, kw, cos, sin, _ = inputs(2, 1, 1, d, "bf16", 5)
    cache = kv4.Kv4Cache.empty(1, 1, 16, d)
    q, k, v = kv4.rope_kv4_append(qkv, cache, torch.arange(2).cuda(), 1, cos=cos, sin=sin,
                                  positions=torch.tensor([3, 4096]).cuda(), q_norm=qw, k_norm=kw, eps=0.0, values=True)
    assert nat.device_status(reset=True) == 2
    assert (q[0] != 0).any() and all((t[1] == 0).all() for t in (q, k, v))
    assert (cache.k_params[0, 0, 0] != 0).any() and (cache.k_params[0, 0, 1:] == 0).all()
