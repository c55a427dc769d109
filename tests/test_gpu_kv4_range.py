"""Values of unlike size in one cache: each group of channels keeps its own precision, whatever the others
hold, and tokens keep theirs beside a token that is far larger, whether the row gives it no weight or
does not see it.

Bar, a channel: the kernels round a value and a probability to fp16 once each (2^-11 of it at most) and
the many-row kernel a key too, which moves a score by at most d = 2^-11 scale sum|q k| and an output by
2 d sum p|v|; fp32 sums are within 1e-4 of sum p|v|; one rounding of the output. Every term goes by the
channel's own sum p|v|.
"""

from __future__ import annotations

import pytest
import torch

import kv4_reference as ref
from conftest import require_b200
from qtts_b200 import _native as nat
from qtts_b200 import kv4
from test_gpu_kv4 import UNIT, filled_cache, request_rows

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(autouse=True)
def _device():
    require_b200()
    nat.device_status(reset=True)
    yield
    torch.cuda.synchronize()
    assert nat.device_status(reset=True) == 0


def check(cache, q, length, name):
    pages = cache.pages
    table = torch.arange(pages, dtype=torch.int32).cuda()[None]
    out = kv4.kv4_attention(q, cache, table, torch.tensor([length], dtype=torch.int32).cuda()).double()
    k, v = request_rows(cache, table[0], length)
    n, sc = q.shape[0], q.shape[2] ** -0.5
    sees = length - n + torch.arange(n, device="cuda") + 1
    want, mag, most = ref.attention(q.double(), k, v, sees, sc)
    bound = (2 * 2.0**-11 + 2 * 2.0**-11 * sc * most[..., None] + 1e-4) * mag + UNIT[name] * want.abs() + 2.0**-24
    ratio = ((out - want).abs() / bound).flatten(0, 1).amax(0)
    assert (ratio <= 1).all(), [f"{x:.3g}" for x in ratio.unflatten(0, (-1, 32)).amax(-1).tolist()]


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [1, 3, 300])
@pytest.mark.parametrize("small", [6, 10, 14])
def test_groups_of_unlike_size(name, d, q_len, small):
    g = torch.Generator().manual_seed(small)
    cache = filled_cache(8, 2, 64, d, g)
    lift = 2.0 ** -torch.tensor([0.0, small, small / 2, small][: d // 32]).cuda()[:, None]
    cache.v_params.copy_(cache.v_params.float() * lift * (1.0 if name == "bf16" else 2.0**7))
    q = torch.randn(q_len, 4, d, generator=g).to(DTYPES[name]).cuda()
    check(cache, q, 500, name)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [1, 4, 300])
@pytest.mark.parametrize("where", ["weightless", "unseen"])
@pytest.mark.parametrize("large", [8, 14])
def test_tokens_beside_a_much_larger_one(d, q_len, where, large):
    g = torch.Generator().manual_seed(large)
    cache = filled_cache(8, 2, 64, d, g)
    q = torch.randn(q_len, 4, d, generator=g).to(torch.bfloat16).cuda()
    if where == "weightless":  # its key turns every query away: exp(-60) and less
        q = q.abs()
        at = 130
        cache.k_params[at // 64, :, at % 64, :, 0] = 0.0
        cache.k_params[at // 64, :, at % 64, :, 1] = -20.0
    else:  # the last token: only the last row sees it, and is left out below
        at = 499
    cache.v_params[at // 64, :, at % 64] *= 2.0**large
    if where == "unseen" and q_len == 1:
        pytest.skip("one new token sees all")
    if where == "weightless":
        check(cache, q, 500, "bf16")
        return
    table = torch.arange(8, dtype=torch.int32).cuda()[None]
    lengths = torch.tensor([500], dtype=torch.int32).cuda()
    out = kv4.kv4_attention(q, cache, table, lengths).double()[:-1]
    k, v = request_rows(cache, table[0], 500)
    sc = d**-0.5
    sees = 500 - q_len + torch.arange(q_len, device="cuda") + 1
    want, mag, most = (t[:-1] for t in ref.attention(q.double(), k, v, sees, sc))
    bound = (2 * 2.0**-11 + 2 * 2.0**-11 * sc * most[..., None] + 1e-4) * mag + UNIT["bf16"] * want.abs()
    assert ((out - want).abs() <= bound).all(), ((out - want).abs() / bound).max()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [1, 300])
@pytest.mark.parametrize("lift", [-12, -8, 0, 5])
def test_fp16_activations_over_small_and_large_values(d, q_len, lift):
    # Scales far below and values near the top of fp16's range; the scores' scale makes up for the keys.
    g = torch.Generator().manual_seed(20 + lift)
    cache = filled_cache(8, 2, 64, d, g)
    for p in (cache.k_params, cache.v_params):
        p.mul_(2.0**lift)
    q = (torch.randn(q_len, 4, d, generator=g) * 2.0**-lift).to(torch.float16).cuda()
    check(cache, q, 500, "fp16")


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [1, 200])
@pytest.mark.parametrize("small", [6, 10, 14])
def test_groups_of_unlike_size_where_nothing_averages(name, d, q_len, small):
    # The first row sees one token, the next ones few: an output is a value, or nearly.
    g = torch.Generator().manual_seed(40 + small)
    cache = filled_cache(8, 2, 64, d, g)
    lift = 2.0 ** -torch.tensor([0.0, small, small / 2, small][: d // 32]).cuda()[:, None]
    cache.v_params.copy_(cache.v_params.float() * lift * (1.0 if name == "bf16" else 2.0**7))
    q = torch.randn(q_len, 4, d, generator=g).to(DTYPES[name]).cuda()
    check(cache, q, q_len, name)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [1, 300])
@pytest.mark.parametrize("lift", [-20, -16, -12])
def test_fp16_activations_over_keys_below_the_range_of_fp16(d, q_len, lift):
    # Scales of keys that fp16 only has as subnormals, with a softmax scale that makes up for them.
    g = torch.Generator().manual_seed(60 + lift)
    cache = filled_cache(8, 2, 64, d, g)
    cache.k_params.mul_(2.0**lift)
    q = torch.randn(q_len, 4, d, generator=g).to(torch.float16).cuda()
    table = torch.arange(8, dtype=torch.int32).cuda()[None]
    sc = d**-0.5 * 2.0**-lift
    out = kv4.kv4_attention(q, cache, table, torch.tensor([500], dtype=torch.int32).cuda(), scale=sc).double()
    k, v = request_rows(cache, table[0], 500)
    sees = 500 - q_len + torch.arange(q_len, device="cuda") + 1
    want, mag, most = ref.attention(q.double(), k, v, sees, sc)
    bound = (2 * 2.0**-11 + 2 * 2.0**-11 * sc * most[..., None] + 1e-4) * mag + UNIT["fp16"] * want.abs()
    assert ((out - want).abs() <= bound).all(), ((out - want).abs() / bound).max()
