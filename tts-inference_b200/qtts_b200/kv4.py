"""The key/value cache in 4 bits: writing it behind the fused projection, attending over it.

A decoder layer's path between its qkv and its output projection
(qtts/models/talker.py:94-136, qtts/layers/rope.py:23-72, the SDPA backend of
qtts/attention/backends/torch_sdpa.py:16-69) as two launches:

* :func:`rope_kv4_append` -- per-head RMSNorm, rotary positions with one to four axes,
  q handed on in its own type, k and v written to the cache in 4 bits;
* :func:`kv4_attention` -- attention of one or many new tokens a request over that cache.

:class:`Kv4Cache` holds the four tensors; ``include/qtts_b200.h`` gives their layout.
Both functions launch on ``torch.cuda.current_stream()`` and never synchronize, so a decode
step with them can be captured in a CUDA graph. They allocate their outputs, a workspace
where a long cache is split among many CTAs, and copies of inputs whose rows are not
16-byte aligned or whose strides the kernels do not take.
There is no CPU path. Indices that live on the device (slots, positions, page numbers,
lengths) are checked by the kernels: one out of range is left out and recorded
(``_native.device_status()``).
"""

from __future__ import annotations

import math

import torch

from . import _native as nat
from .quant.kernels import _flags, _require_cuda

GROUP = 32  # channels that share a scale and a minimum
HEAD_DIMS = (64, 128)
_HALVES = (32, 64)
_DTYPES = {torch.bfloat16: nat.BF16, torch.float16: nat.FP16}
_SCALES = {d: 1.0 / math.sqrt(d) for d in HEAD_DIMS}
_SPLIT_FROM = 897  # tokens: eight steps of 128, which two CTAs may share


class Kv4Cache:
    """A paged key/value cache in 4 bits.

    ``k_codes`` / ``v_codes`` uint8 ``[pages, kv_heads, page_size, head_dim / 2]`` and
    ``k_params`` / ``v_params`` bf16 ``[pages, kv_heads, page_size, head_dim / 32, 2]``
    (scale, minimum), all contiguous: 5 bits a channel in all. ``page_size`` is a
    multiple of 16. A slot cache is one page a request.
    """

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params", "pages", "kv_heads", "page_size", "head_dim", "_ptrs",
                 "_index")

    def __init__(self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor,
                 v_params: torch.Tensor) -> None:
        shape = k_codes.shape
        if len(shape) != 4 or v_codes.shape != shape or k_codes.dtype is not torch.uint8 or \
                v_codes.dtype is not torch.uint8:
            raise ValueError("codes must be uint8 [pages, kv_heads, page_size, head_dim / 2], keys and values alike")
        pages, kv_heads, page_size, half = shape
        if half not in _HALVES:
            raise ValueError(f"head_dim {2 * half}: the 4-bit cache takes {HEAD_DIMS}")
        if kv_heads < 1:
            raise ValueError("kv_heads is at least 1")
        if page_size < 16 or page_size % 16:
            raise ValueError(f"page_size {page_size} is not a multiple of 16")
        want = (pages, kv_heads, page_size, half * 2 // GROUP, 2)
        if k_params.shape != want or v_params.shape != want or k_params.dtype is not torch.bfloat16 or \
                v_params.dtype is not torch.bfloat16:
            raise ValueError(f"params must be bf16 {want}, keys and values alike")
        if not (k_codes.is_contiguous() and k_params.is_contiguous() and v_codes.is_contiguous()
                and v_params.is_contiguous()):
            raise ValueError("the cache's tensors must be contiguous")
        index = k_codes.get_device()
        if not index == k_params.get_device() == v_codes.get_device() == v_params.get_device():
            raise ValueError("the cache's tensors must be on one device")
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, kv_heads, page_size, 2 * half
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self._index = index
        self._ptrs = (k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(), pages,
                      page_size)

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
    are the weights of the per-head RMSNorm. The codes stored are those of the same steps as
    separate fp32 torch operations, bit for bit.

    Returns q ``[tokens, q_heads, head_dim]``; with ``values`` also the keys and values
    ``[tokens, kv_heads, head_dim]`` as the cache will give them back.
    """
    kv_heads, d = cache.kv_heads, cache.head_dim
    width = (q_heads + 2 * kv_heads) * d
    if qkv.dim() != 2 or qkv.shape[1] != width:
        raise ValueError(f"qkv is {tuple(qkv.shape)}, expected [tokens, {width}]")
    dtype = _DTYPES.get(qkv.dtype)
    if dtype is None:
        raise TypeError(f"qkv must be bf16 or fp16, got {qkv.dtype}")
    tokens = qkv.shape[0]
    if slots.dtype is not torch.int64 or slots.shape != (tokens,) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 [{tokens}]")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin are given together")
    index = qkv.get_device()
    if index < 0 or cache._index != index or slots.get_device() != index:
        _require_cuda(qkv, cache.k_codes, slots)
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    axes = table_len = ldpos = 0
    cos_ptr = sin_ptr = pos_ptr = None
    if cos is not None:
        if positions is None:
            raise ValueError("positions are needed with cos and sin")
        if positions.dtype is not torch.int64 or positions.dim() not in (1, 2) or positions.shape[-1] != tokens or \
                (tokens > 1 and positions.stride(-1) != 1):
            raise ValueError(f"positions must be int64 [axes, {tokens}] with unit stride along the tokens")
        axes = positions.shape[0] if positions.dim() == 2 else 1
        sections = (d // 2,) if sections is None else tuple(sections)
        if len(sections) != axes or not 1 <= axes <= 4 or sum(sections) != d // 2 or min(sections) < 0:
            raise ValueError(f"sections {sections} do not share {d // 2} pairs among {axes} axes")
        table_shape = cos.shape
        if len(table_shape) != 2 or table_shape[1] != d // 2 or sin.shape != table_shape or \
                cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or not cos.is_contiguous() or \
                not sin.is_contiguous():
            raise ValueError(f"cos and sin must be contiguous fp32 [length, {d // 2}]")
        if cos.get_device() != index or sin.get_device() != index or positions.get_device() != index:
            _require_cuda(qkv, cos, sin, positions)
        table_len = table_shape[0]
        ldpos = tokens if axes == 1 else positions.stride(0)
        if ldpos < tokens:  # an axis that is broadcast
            positions = positions.contiguous()
            ldpos = tokens
        cos_ptr, sin_ptr, pos_ptr = cos.data_ptr(), sin.data_ptr(), positions.data_ptr()
    if q_norm is not None:
        q_norm = _norm_weight(q_norm, d, qkv)
    if k_norm is not None:
        k_norm = _norm_weight(k_norm, d, qkv)
    q = qkv.new_empty((tokens, q_heads, d))
    k_ptr = v_ptr = None
    if values:
        k_values = qkv.new_empty((tokens, kv_heads, d))
        v_values = torch.empty_like(k_values)
        k_ptr, v_ptr = k_values.data_ptr(), v_values.data_ptr()
    nat.launch(
        "qtts_rope_kv4_append", index, qkv.data_ptr(), qkv.stride(0) if tokens > 1 else width, dtype, tokens, q_heads,
        kv_heads, d, None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps,
        cos_ptr, sin_ptr, table_len, pos_ptr, ldpos, axes, sections if axes else None, interleaved, slots.data_ptr(), q.data_ptr(),
        q_heads * d, *cache._ptrs, k_ptr, v_ptr, _flags())
    return (q, k_values, v_values) if values else q


def _norm_weight(w: torch.Tensor, d: int, qkv: torch.Tensor) -> torch.Tensor:
    if w.shape != (d,) or w.dtype is not qkv.dtype:
        raise ValueError(f"a norm weight must be {qkv.dtype} [{d}]")
    if w.get_device() != qkv.get_device():
        _require_cuda(qkv, w)
    if w.stride(0) != 1 or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    return w


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
    says how many at most (rows of no request keep what ``out`` held: in a new ``out``,
    anything). The new tokens are the last ones of their request: with
    ``causal`` each sees the tokens up to itself, without it every cached token (cross
    attention to an encoder's states, for instance). ``q_heads`` is a multiple of the
    cache's heads. A row that sees nothing gives zeros. ``scale`` defaults to
    ``1 / sqrt(head_dim)``. Returns ``[total, q_heads, head_dim]``.
    """
    shape = q.shape
    kv_heads, d = cache.kv_heads, cache.head_dim
    if len(shape) != 3 or shape[2] != d or shape[1] % kv_heads or not shape[1]:
        raise ValueError(f"q is {tuple(shape)}, expected [tokens, a multiple of {kv_heads}, {d}]")
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise TypeError(f"q must be bf16 or fp16, got {q.dtype}")
    total, heads = shape[0], shape[1]
    if lengths.dtype is not torch.int32 or lengths.dim() != 1 or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 [batch]")
    batch = lengths.shape[0]
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch or \
            (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError(f"block_table must be int32 [{batch}, columns] with unit stride along the columns")
    columns = block_table.shape[1]
    starts_ptr = None
    index = q.get_device()
    if q_starts is None:
        max_q = total // batch if batch else 0
        if max_q * batch != total:
            raise ValueError(f"{total} tokens do not share evenly among {batch} requests: give q_starts")
    else:
        if q_starts.dtype is not torch.int32 or q_starts.shape != (batch + 1,) or not q_starts.is_contiguous():
            raise ValueError(f"q_starts must be a contiguous int32 [{batch + 1}]")
        if max_q is None:
            raise ValueError("max_q is needed with q_starts")
        if max_q > total:
            max_q = total
        if q_starts.get_device() != index:
            _require_cuda(q, q_starts)
        starts_ptr = q_starts.data_ptr()
    if scale is None:
        scale = _SCALES[d]
    elif not 0.0 < scale < math.inf:
        raise ValueError(f"scale {scale} is not positive and finite")
    if index < 0 or cache._index != index or block_table.get_device() != index or lengths.get_device() != index:
        _require_cuda(q, cache.k_codes, block_table, lengths)
    dense = q.is_contiguous()
    if dense:
        token_stride, head_stride = heads * d, d
    else:
        token_stride, head_stride = q.stride(0), q.stride(1)
        if q.stride(2) != 1 or token_stride % 8 or head_stride % 8 or head_stride < d:
            q = q.contiguous()
            token_stride, head_stride = heads * d, d
    q_ptr = q.data_ptr()
    if q_ptr % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        q_ptr, token_stride, head_stride = q.data_ptr(), heads * d, d
    if out is None:
        out = torch.empty_like(q) if dense else q.new_empty(shape)
    elif out.shape != shape or out.dtype is not q.dtype or not out.is_contiguous() or out.get_device() != index:
        raise ValueError(f"out must be a contiguous {q.dtype} {tuple(shape)} on q's device")
    work_ptr = None
    tokens = columns * cache.page_size
    if tokens >= _SPLIT_FROM:  # fewer tokens are never split across a workspace
        need = nat.lib().qtts_kv4_attention_workspace(total, max_q, batch, heads, kv_heads, d, tokens)
        if need:
            workspace = q.new_empty(need, dtype=torch.uint8)
            work_ptr = workspace.data_ptr()
    nat.launch(
        "qtts_kv4_attention", index, q_ptr, token_stride, head_stride, dtype, *cache._ptrs, block_table.data_ptr(),
        block_table.stride(0) if batch > 1 else columns, columns, lengths.data_ptr(), starts_ptr, total, max_q, batch,
        heads, kv_heads, d, scale, causal, out.data_ptr(), heads * d, work_ptr, _flags())
    return out
