"""Rows of q that belong to no request (a padded total, as a captured graph has; a first row above
0) keep what `out` held, bit for bit, whether the call is split across a workspace or not, and rows of
requests do not depend on them."""

from __future__ import annotations

import pytest
import torch

from conftest import require_b200
from qtts_b200 import _native as nat
from qtts_b200 import kv4
from test_gpu_kv4 import filled_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    require_b200()
    nat.device_status(reset=True)
    yield
    torch.cuda.synchronize()
    assert nat.device_status(reset=True) == 0


def workspace(total, max_q, batch, heads, kv_heads, d, tokens):
    return nat.lib().qtts_kv4_attention_workspace(total, max_q, batch, heads, kv_heads, d, tokens)


CASES = [  # new tokens a request, tokens of the table, whether that splits through the workspace
    ([1, 1], 128, False), ([1, 1], 8192, True), ([1, 0, 1], 8192, True), ([1], 65536, True), ([3, 2], 128, False),
    ([3, 2], 8192, True), ([200], 512, False), ([200, 0, 70], 4096, True),
]


@pytest.mark.parametrize("news,tokens,split", CASES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("front,back", [(0, 5), (4, 0), (3, 7)])
def test_rows_of_no_request_are_not_written(news, tokens, split, d, front, back):
    g = torch.Generator().manual_seed(tokens + front)
    heads, kv_heads, page = 4, 2, 64
    batch, used = len(news), sum(news)
    cache = filled_cache(64, kv_heads, page, d, g)
    table = torch.randint(0, 64, (batch, tokens // page), generator=g).to(torch.int32).cuda()
    lengths = torch.tensor([min(tokens, 1500) - 31 * b for b in range(batch)], dtype=torch.int32).clamp_min(64).cuda()
    starts = torch.tensor([front + sum(news[:b]) for b in range(batch + 1)], dtype=torch.int32).cuda()
    total, max_q = front + used + back, max(news)
    assert (workspace(total, max_q, batch, heads, kv_heads, d, tokens) > 0) == split
    q = torch.randn(total, heads, d, generator=g).to(torch.bfloat16).cuda()
    # Whatever the caching allocator hands out as a workspace has been used before.
    junk = torch.full((64 << 20,), 7.0, device="cuda")
    del junk
    out = torch.full_like(q, 3.5)
    kv4.kv4_attention(q, cache, table, lengths, q_starts=starts, max_q=max_q, out=out)
    assert (out[:front] == 3.5).all() and (out[front + used:] == 3.5).all()
    assert (out[front : front + used] != 3.5).any()
    tight = kv4.kv4_attention(q[front : front + used].contiguous(), cache, table, lengths, q_starts=starts - front,
                              max_q=max_q)
    assert torch.equal(tight, out[front : front + used])


@pytest.mark.parametrize("tokens", [128, 8192])
def test_a_refused_request_is_recorded_and_not_written(tokens):
    # The second request brings more tokens than max_q says; the first and the third are answered.
    g = torch.Generator().manual_seed(2)
    cache = filled_cache(8, 2, 64, 128, g)
    table = torch.randint(0, 8, (3, tokens // 64), generator=g).to(torch.int32).cuda()
    lengths = torch.tensor([100, 90, 80], dtype=torch.int32).cuda()
    q = torch.randn(4, 4, 128, generator=g).to(torch.bfloat16).cuda()
    out = torch.full_like(q, 3.5)
    kv4.kv4_attention(q, cache, table, lengths, q_starts=torch.tensor([0, 1, 3, 4], dtype=torch.int32).cuda(), max_q=1,
                      out=out)
    assert nat.device_status(reset=True) == 2
    assert (out[1:3] == 3.5).all() and (out[0] != 3.5).any() and (out[3] != 3.5).any()
    one = kv4.kv4_attention(q[:1].contiguous(), cache, table[:1], lengths[:1])
    assert torch.allclose(out[:1].float(), one.float(), atol=2**-7)
