"""The 4-bit cache, its writer and its attention in float64, from the formulas alone."""

from __future__ import annotations

import math

import torch

GROUP = 32


def nibble_of(d: int, keys: bool) -> torch.Tensor:
    """Position in a row of each channel's code, counted in nibbles from the row's start."""
    n, run = d // GROUP, 8 if keys else 4
    place = torch.empty(d, dtype=torch.int64)
    for ch in range(d):
        j, rest = divmod(ch, GROUP)
        word, i = divmod(rest, run)
        place[ch] = (word * n + j) * run + i
    return place


def read_rows(codes: torch.Tensor, params: torch.Tensor, keys: bool) -> torch.Tensor:
    """uint8 [..., D/2] and bf16 [..., D/32, 2] -> float64 [..., D]."""
    d = codes.shape[-1] * 2
    place = nibble_of(d, keys).to(codes.device)
    byte = codes[..., place // 2].to(torch.int64)
    code = (byte >> (4 * (place % 2))) & 15
    p = params.double()[..., torch.arange(d, device=codes.device) // GROUP, :]
    return code.double() * p[..., 0] + p[..., 1]


def write_rows(x: torch.Tensor, keys: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """float64 [..., D] -> (uint8 [..., D/2], bf16 [..., D/32, 2])."""
    d = x.shape[-1]
    g = x.unflatten(-1, (-1, GROUP))
    scale = ((g.amax(-1) - g.amin(-1)) / 15).to(torch.bfloat16)
    low = g.amin(-1).to(torch.bfloat16)
    s = scale.double()[..., None]
    code = torch.where(s > 0, (g - low.double()[..., None]) / s.clamp_min(1e-300), torch.zeros_like(g))
    code = code.round().clamp(0, 15).flatten(-2).to(torch.uint8)
    flat = torch.empty_like(code)
    flat[..., nibble_of(d, keys).to(x.device)] = code
    return flat[..., 0::2] | (flat[..., 1::2] << 4), torch.stack((scale, low), -1)


def attention(q, k, v, sees, scale):
    """q [n, H, D], k and v [L, Hkv, D] float64, sees [n] -> out, sum of p|v|, and the largest
    sum over channels of |q k| of a seen token (for error bounds), each [n, H, D] or [n, H]."""
    n, heads, d = q.shape
    share = heads // k.shape[1]
    out = torch.zeros_like(q)
    mag = torch.zeros_like(q)
    most = torch.zeros(n, heads, dtype=torch.float64, device=q.device)
    for h in range(heads):
        kh, vh = k[:, h // share], v[:, h // share]
        late = torch.arange(k.shape[0], device=q.device)[None, :] >= sees[:, None]
        score = (q[:, h] @ kh.T * scale).masked_fill(late, -math.inf)
        some = sees > 0
        p = torch.zeros_like(score)
        p[some] = torch.softmax(score[some], -1)
        out[:, h], mag[:, h] = p @ vh, p @ vh.abs()
        most[:, h] = (q[:, h].abs() @ kh.abs().T).masked_fill(late, 0).amax(-1) if k.shape[0] else 0
    return out, mag, most
