"""Residual addition + RMSNorm + 8-bit quantization in one launch, against float64.

Bars, from the arithmetic: the residual is one fp32 addition and one rounding, equal bit for bit
to torch's; the scale is a maximum of fp32 values, each some ulps off (the sum of W squares in
any order: W * 2^-24 at the very worst, far less in a tree): 1e-5; a code stands for y within
half a step: scale / 2 for int8; 2^-4 |y| or 2^-10 scale (below the smallest normal) for e4m3;
with 1e-4 of the row's scale-range on top for the fp32 steps before the rounding."""

from __future__ import annotations

import pytest
import torch

from conftest import require_b200
from qtts_b200 import _native as nat
from qtts_b200.quant import kernels as qk

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


@pytest.fixture(autouse=True)
def _device():
    require_b200()
    nat.device_status(reset=True)
    yield
    torch.cuda.synchronize()
    assert nat.device_status() == 0


def check(x, r, w, eps, to, **kw):
    x0, r0 = x.clone(), r.clone() if r is not None else None
    q, scale, h = qk.add_rms_norm_quant(x, r, w, eps, dtype=to, **kw)
    width = x.shape[-1]
    rows = x.numel() // width
    assert q.shape == (rows, width) and q.dtype == to and scale.shape == (rows, 1)
    total = x0.double()
    if r is not None:
        assert torch.equal(h, (x0.float() + r0.float()).to(x.dtype)) and h.shape == x.shape
        total = (x0.float() + r0.float()).double()
    else:
        assert h is None
    total = total.reshape(rows, width)
    y = w.double() * total / (total.square().mean(-1, keepdim=True) + eps).sqrt()
    most = 127 if to == torch.int8 else 448
    want = y.abs().amax(-1, keepdim=True).clamp_min(1e-6) / most
    assert ((scale.double() - want).abs() <= 1e-5 * want).all()
    s = scale.double()
    err = (q.double() * s - y).abs()
    half = 0.5 * s if to == torch.int8 else torch.maximum(2.0**-4 * y.abs(), 2.0**-10 * s)
    assert (err <= half * (1 + 1e-4) + 1e-4 * want).all()
    if to == torch.int8:
        assert (q.abs().amax(-1) <= 127).all() and (q.int().amin() >= -127)


@pytest.mark.parametrize("name", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("to", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("width", [1, 7, 64, 1000, 1024, 2048, 2049, 6144, 8192, 16392, 40000])
def test_against_float64(name, to, width):
    g = torch.Generator().manual_seed(width)
    x = (0.5 * torch.randn(5, width, generator=g)).to(DTYPES[name]).cuda()
    r = (2.0 * torch.randn(5, width, generator=g)).to(DTYPES[name]).cuda()
    w = (1 + 0.2 * torch.randn(width, generator=g)).to(DTYPES[name]).cuda()
    x[1], r[1] = 0, 0
    x[2], r[2] = x[2] * 1e-3, r[2] * 1e-3
    check(x, r, w, 1e-6, to)
    check(x, None, w, 1e-5, to)


@pytest.mark.parametrize("rows", [1, 2, 3, 33, 257, 1500])
@pytest.mark.parametrize("width", [512, 2048, 5120])
def test_row_counts(rows, width):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, width, generator=g).to(torch.bfloat16).cuda()
    r = torch.randn(rows, width, generator=g).to(torch.bfloat16).cuda()
    w = torch.ones(width, dtype=torch.bfloat16).cuda()
    check(x, r, w, 1e-6, torch.float8_e4m3fn)
    check(x, r, w, 1e-6, torch.int8)


def test_shapes_strides_and_in_place():
    g = torch.Generator().manual_seed(1)
    w = (1 + 0.2 * torch.randn(640, generator=g)).to(torch.bfloat16).cuda()
    wide = torch.randn(6, 1283, generator=g).to(torch.bfloat16).cuda()
    check(wide[:, :640], wide[:, 643:1283], w, 1e-6, torch.float8_e4m3fn)  # rows on 2-byte boundaries
    even = torch.randn(6, 1280, generator=g).to(torch.bfloat16).cuda()
    check(even[:, :640], even[:, 640:], w, 1e-6, torch.int8)
    x3 = torch.randn(2, 3, 640, generator=g).to(torch.bfloat16).cuda()
    r3 = torch.randn(2, 3, 640, generator=g).to(torch.bfloat16).cuda()
    check(x3, r3, w, 1e-6, torch.float8_e4m3fn)
    r_in = r3.clone()
    check(x3, r_in, w, 1e-6, torch.float8_e4m3fn, residual_out=r_in)
    empty = torch.empty(0, 640, dtype=torch.bfloat16).cuda()
    q, s, h = qk.add_rms_norm_quant(empty, empty, w)
    assert q.shape == (0, 640) and s.shape == (0, 1) and h.shape == (0, 640)


@pytest.mark.parametrize("to", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("width", [640, 641, 20000])
def test_non_finite_rows_are_marked(to, bad, width):
    x = torch.randn(3, width, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    x[1, 17] = bad
    w = torch.ones(width, dtype=torch.bfloat16).cuda()
    _, scale, h = qk.add_rms_norm_quant(x, torch.zeros_like(x), w, dtype=to)
    assert torch.isnan(scale[1]).all() and torch.isfinite(scale[[0, 2]]).all()
    assert torch.equal(h.isfinite(), x.isfinite())


def test_feeds_the_linears():
    g = torch.Generator().manual_seed(3)
    m, k, n = 9, 2048, 512
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).cuda()
    r = torch.randn(m, k, generator=g).to(torch.bfloat16).cuda()
    w = (1 + 0.1 * torch.randn(k, generator=g)).to(torch.bfloat16).cuda()
    lin = (torch.randn(n, k, generator=g) * 0.02).to(torch.bfloat16).cuda()
    h = x.double() + r.double()
    want = (w.double() * h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt()) @ lin.double().T
    q, s, _ = qk.add_rms_norm_quant(x, r, w)
    wq, ws = qk.quantize_fp8_rows(lin)
    y = qk.fp8_scaled_mm(q, s, wq, ws, None, torch.bfloat16)
    # e4m3 on both sides: 2^-4 / sqrt(3) rms an operand, which average out over K products.
    assert (y.double() - want).norm() <= 0.06 * want.norm()
    q, s, _ = qk.add_rms_norm_quant(x, r, w, dtype=torch.int8)
    wq, ws = qk.quantize_int8_rows(lin)
    y = qk.i8_scaled_mm(q, s, wq, ws, None, torch.bfloat16)
    assert (y.double() - want).norm() <= 0.03 * want.norm()
