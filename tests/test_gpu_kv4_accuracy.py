"""How near the attention over the 4-bit cache comes to 64 bits, all outputs of a call together.

Bar, from the roundings (2-norm of the error over that of the result): rounding to p significant bits
is off by at most 2^-p of a value and, evenly spread, by 2^(1-p) / sqrt(12) of it in the mean square at
worst (a value just above a power of two). The output is rounded once (bf16: 2.26e-3, fp16: 2.82e-4);
probabilities, values and, through the scores, keys are rounded to fp16 at most once each (2.82e-4 each;
a key's rounding moves a score of order one by no more). Independent, together: 2.31e-3 and 5.64e-4, and
4 % for the spread of a call's own sum and fp32: 2.4e-3 and 5.9e-4. bf16 operands (2.26e-3 each)
would not pass.
"""

from __future__ import annotations

import pytest
import torch

import kv4_reference as ref
from conftest import require_b200
from qtts_b200 import _native as nat
from qtts_b200 import kv4
from test_gpu_kv4 import filled_cache, request_rows

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BAR = {"bf16": 2.4e-3, "fp16": 5.9e-4}


@pytest.fixture(autouse=True)
def _device():
    require_b200()
    nat.device_status(reset=True)
    yield
    torch.cuda.synchronize()
    assert nat.device_status(reset=True) == 0


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,q_len", [([513, 500, 31], 1), ([4096, 2000], 1), ([700, 650], 5), ([300, 900], 40),
                                           ([512, 480], 300), ([2000], 200)])
def test_error_against_64_bits(name, d, causal, lengths, q_len):
    g = torch.Generator().manual_seed(lengths[0] + q_len)
    heads, kv_heads, page = 8, 4, 32
    columns = -(-max(lengths) // page)
    cache = filled_cache(len(lengths) * columns, kv_heads, page, d, g)
    table = torch.randperm(len(lengths) * columns, generator=g).to(torch.int32).view(-1, columns).cuda()
    q = torch.randn(len(lengths) * q_len, heads, d, generator=g).to(DTYPES[name]).cuda()
    out = kv4.kv4_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32).cuda(),
                            causal=causal).double()
    err2 = ref2 = 0.0
    for b, n in enumerate(lengths):
        k, v = request_rows(cache, table[b], n)
        i = torch.arange(q_len, device="cuda")
        sees = n - q_len + i + 1 if causal else torch.full((q_len,), n, device="cuda")
        rows = slice(b * q_len, (b + 1) * q_len)
        want, _, _ = ref.attention(q[rows].double(), k, v, sees, d**-0.5)
        err2 += (out[rows] - want).square().sum().item()
        ref2 += want.square().sum().item()
    assert err2 <= BAR[name] ** 2 * ref2, f"{(err2 / ref2) ** 0.5:.2e}"
