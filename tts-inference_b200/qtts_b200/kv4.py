"""The key/value cache in 4 bits: writing it behind the fused projection, attending over it.

A decoder layer's path between its qkv and its output projection
(qtts/models/talker.py:94-136, qtts/layers/rope.py:23-72, the SDPA backend of
qtts/attention/backends/torch_sdpa.py:16-69) as two launches:

* :func:`rope_kv4_append` -- per-head RMSNorm, rotary positions with one to four axes,
  q handed on in its own type, k and v written to the cache in 4 bits;
* :func:`kv4_attention` -- attention of one or many new tokens a request over that cache.

:class:`Kv4Cache` holds the four tensors; ``include/qtts_b200.h`` gives their layout.
Both functions launch on ``torch.cuda.current_stream()``, allocate only their outputs
and never synchronize, so a decode step with them can be captured in a CUDA graph.
There is no CPU path. Indices that live on the device (slots, positions, page numbers,
lengths) are checked by the kernels: one out of range is left out and recorded
(``_native.device_status()``).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as nat
from .quant.kernels import _flags, _require_cuda

GROUP = 32  # channels that share a scale and a minimum
HEAD_DIMS = (64, 128)


class Kv4Cache:
    """A paged key/value cache in 4 bits.

    ``k_codes`` / ``v_codes`` uint8 ``[pages, kv_heads, page_size, head_dim / 2]`` and
    ``k_params`` / ``v_params`` bf16 ``[pages, kv_heads, page_size, head_dim / 32, 2]``
    (scale, minimum), all contiguous: 5 bits a channel in all. ``page_size`` is a
    multiple of 16. A slot cache is one page a request.
    """

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params", "pages", "kv_heads", "page_size", "head_dim", "_ptrs")

    def __init__(self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor,
                 v_params: torch.Tensor) -> None:
        shape = k_codes.shape
        if len(shape) != 4 or v_codes.shape != shape or k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8:
            raise ValueError("codes must be uint8 [pages, kv_heads, page_size, head_dim / 2], keys and values alike")
        self.pages, self.kv_heads, self.page_size, half = shape
        self.head_dim = 2 * half
        if self.head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim {self.head_dim}: the 4-bit cache takes {HEAD_DIMS}")
        if self.page_size < 16 or self.page_size % 16:
            raise ValueError(f"page_size {self.page_size} is not a multiple of 16")
        want = (*shape[:3], self.head_dim // GROUP, 2)
        for p in (k_params, v_params):
            if p.shape != want or p.dtype != torch.bfloat16:
                raise ValueError(f"params must be bf16 {want}, got {p.dtype} {tuple(p.shape)}")
        for t in (k_codes, k_params, v_codes, v_params):
            if not t.is_contiguous():
                raise ValueError("the cache's tensors must be contiguous")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self._ptrs = (k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr())

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> Kv4Cache:
        """A new cache (zeroed)."""
        def pair():
            return (torch.zeros(pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device),
                    torch.zeros(pages, kv_heads, page_size, head_dim // GROUP, 2, dtype=torch.bfloat16, device=device))
        return cls(*pair(), *pair())

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_params, self.v_codes, self.v_params))

    def values(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that the cache stands for, fp32 ``[pages, kv_heads, page_size,
        head_dim]`` (torch ops, for inspection)."""
        def one(codes, params, run):
            n = self.head_dim // GROUP
            c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
            c = c.unflatten(-1, (GROUP // run, n, run)).transpose(-3, -2).flatten(-2).float()
            p = params.float()
            return (c * p[..., 0:1] + p[..., 1:2]).flatten(-2)
        return one(self.k_codes, self.k_params, 8), one(self.v_codes, self.v_params, 4)


def rope_kv4_append(
    qkv: torch.Tensor,
    cache: Kv4Cache,
    slots: torch.Tensor,
    q_heads: int,
    *,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    sections: tuple[int, ...] | None = None,
    interleaved: bool = False,
    q_norm: torch.Tensor | None = None,
    k_norm: torch.Tensor | None = None,
    eps: float = 1e-6,
    values: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Norm and turn the heads of ``qkv``, write its keys and values to ``cache`` in 4 bits.

    ``qkv`` is ``[tokens, (q_heads + 2 * kv_heads) * head_dim]`` (bf16 or fp16): q heads,
    k heads, v heads. ``slots`` ``[tokens]`` int64 are the tokens' places in the cache
    (``page * page_size + row``, all different; negative: not stored). With ``cos`` and
    ``sin`` (fp32 tables ``[length, head_dim / 2]``) every pair ``(j, j + head_dim / 2)`` of
    a q or k head is turned by the tables' row ``positions[axis of j]``; ``positions`` is
    ``[tokens]`` or ``[axes, tokens]`` int64, ``sections`` says how many pairs each axis has
    (in order, or taking turns when ``interleaved``). ``q_norm`` / ``k_norm`` ``[head_dim]``
    are the weights of the per-head RMSNorm.

    Returns q ``[tokens, q_heads, head_dim]``; with ``values`` also the keys and values
    ``[tokens, kv_heads, head_dim]`` as the cache will give them back.
    """
    kv_heads, d = cache.kv_heads, cache.head_dim
    width = (q_heads + 2 * kv_heads) * d
    if qkv.dim() != 2 or qkv.shape[1] != width:
        raise ValueError(f"qkv is {tuple(qkv.shape)}, expected [tokens, {width}]")
    if qkv.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"qkv must be bf16 or fp16, got {qkv.dtype}")
    tokens = qkv.shape[0]
    if slots.dtype != torch.int64 or slots.shape != (tokens,) or (tokens > 1 and slots.stride(0) != 1):
        raise ValueError(f"slots must be a contiguous int64 [{tokens}]")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin are given together")
    device = _require_cuda(qkv, cache.k_codes, slots, cos, sin, positions, q_norm, k_norm)
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    axes, table_len, ldpos, section_array, table = 0, 0, 0, None, (None, None, None)
    if cos is not None:
        if positions is None:
            raise ValueError("positions are needed with cos and sin")
        if positions.dim() == 1:
            positions = positions[None]
        axes = positions.shape[0]
        if sections is None:
            sections = (d // 2,)
        if len(sections) != axes or not 1 <= axes <= 4 or sum(sections) != d // 2 or min(sections) < 0:
            raise ValueError(f"sections {tuple(sections)} do not share {d // 2} pairs among {axes} axes")
        if positions.dtype != torch.int64 or positions.shape[1] != tokens or (tokens > 1 and positions.stride(1) != 1):
            raise ValueError(f"positions must be int64 [axes, {tokens}] with unit stride along the tokens")
        for t in (cos, sin):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape != cos.shape or t.shape[1] != d // 2 or \
                    not t.is_contiguous():
                raise ValueError(f"cos and sin must be contiguous fp32 [length, {d // 2}]")
        table_len = cos.shape[0]
        ldpos = max(positions.stride(0), tokens) if axes > 1 else tokens
        section_array = (ctypes.c_int * axes)(*sections)
        table = (cos.data_ptr(), sin.data_ptr(), positions.data_ptr())
    norms = []
    for w in (q_norm, k_norm):
        if w is not None:
            if w.shape != (d,) or w.dtype != qkv.dtype:
                raise ValueError(f"a norm weight must be {qkv.dtype} [{d}]")
            if w.stride(0) != 1 or w.data_ptr() % 16:
                w = w.clone(memory_format=torch.contiguous_format)
        norms.append(w)
    q = torch.empty((tokens, q_heads, d), device=device, dtype=qkv.dtype)
    k_values = v_values = None
    if values:
        k_values = torch.empty((tokens, kv_heads, d), device=device, dtype=qkv.dtype)
        v_values = torch.empty((tokens, kv_heads, d), device=device, dtype=qkv.dtype)
    code = nat.lib().qtts_rope_kv4_append(
        qkv.data_ptr(), qkv.stride(0) if tokens > 1 else width, nat.dtype_code(qkv.dtype), tokens, q_heads, kv_heads, d,
        norms[0].data_ptr() if norms[0] is not None else None, norms[1].data_ptr() if norms[1] is not None else None,
        eps, table[0], table[1], table_len, table[2], ldpos, axes, section_array, int(interleaved), slots.data_ptr(),
        q.data_ptr(), q_heads * d, *cache._ptrs, cache.pages, cache.page_size,
        k_values.data_ptr() if values else None, v_values.data_ptr() if values else None, _flags(),
        nat.stream_ptr(device))
    nat.check(code, "qtts_rope_kv4_append")
    return (q, k_values, v_values) if values else q


def kv4_attention(
    q: torch.Tensor,
    cache: Kv4Cache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    q_starts: torch.Tensor | None = None,
    max_q: int | None = None,
    scale: float | None = None,
    causal: bool = True,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of new tokens over the 4-bit cache they are already in.

    ``q`` is ``[total, q_heads, head_dim]`` (bf16 or fp16, unit stride along the channels),
    ``block_table`` ``[batch, columns]`` int32 page numbers and ``lengths`` ``[batch]`` int32
    the cached tokens of each request, new ones included. Without ``q_starts`` every
    request brings ``total / batch`` new tokens (one, in a decode step); with it, ``[batch +
    1]`` int32, request b brings rows ``q_starts[b]`` to ``q_starts[b + 1]`` and ``max_q``
    says how many at most. The new tokens are the last ones of their request: with
    ``causal`` each sees the tokens up to itself, without it every cached token (cross
    attention to an encoder's states, for instance). ``q_heads`` is a multiple of the
    cache's heads. A row that sees nothing gives zeros. ``scale`` defaults to
    ``1 / sqrt(head_dim)``. Returns ``[total, q_heads, head_dim]``.
    """
    if q.dim() != 3 or q.shape[2] != cache.head_dim or q.shape[1] % cache.kv_heads:
        raise ValueError(f"q is {tuple(q.shape)}, expected [tokens, a multiple of {cache.kv_heads}, {cache.head_dim}]")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bf16 or fp16, got {q.dtype}")
    total, heads, d = q.shape
    batch = lengths.shape[0]
    if lengths.dtype != torch.int32 or lengths.dim() != 1 or (batch > 1 and lengths.stride(0) != 1):
        raise ValueError("lengths must be a contiguous int32 [batch]")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch or \
            (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 [{batch}, columns] with unit stride along the columns")
    if q_starts is None:
        if batch == 0 or total % batch:
            if total:
                raise ValueError(f"{total} tokens do not share evenly among {batch} requests: give q_starts")
        max_q = total // batch if batch else 0
    else:
        if q_starts.dtype != torch.int32 or q_starts.shape != (batch + 1,) or (batch > 0 and q_starts.stride(0) != 1):
            raise ValueError(f"q_starts must be a contiguous int32 [{batch + 1}]")
        if max_q is None:
            raise ValueError("max_q is needed with q_starts")
        max_q = min(max_q, total)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    elif not 0.0 < scale < math.inf:
        raise ValueError(f"scale {scale} is not positive and finite")
    device = _require_cuda(q, cache.k_codes, block_table, lengths, q_starts, out)
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.stride(1) < d or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty((total, heads, d), device=device, dtype=q.dtype)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {q.dtype} {tuple(q.shape)}")
    columns = block_table.shape[1]
    need = nat.lib().qtts_kv4_attention_workspace(total, max_q, batch, heads, cache.kv_heads, d,
                                                  columns * cache.page_size)
    workspace = torch.empty(need, device=device, dtype=torch.uint8) if need else None
    code = nat.lib().qtts_kv4_attention(
        q.data_ptr(), q.stride(0), q.stride(1), nat.dtype_code(q.dtype), *cache._ptrs, cache.pages, cache.page_size,
        block_table.data_ptr(), block_table.stride(0) if batch > 1 else columns, columns, lengths.data_ptr(),
        q_starts.data_ptr() if q_starts is not None else None, total, max_q, batch, heads, cache.kv_heads, d,
        scale, int(causal), out.data_ptr(), heads * d,
        workspace.data_ptr() if need else None, _flags(), nat.stream_ptr(device))
    nat.check(code, "qtts_kv4_attention")
    return out
