"""The 4-bit key/value cache on the GPU: the fused norm + rotary + cache write and the attention
over the cache, against float64 (kv4_reference).

Bars, from the arithmetic:
* q of the writer: one rounding to its type after fp32 steps: |err| <= u |ref| + 1e-5 of the
  row's largest magnitude (u, half a step: 2^-8 for bf16's 8 significant bits, 2^-11 for fp16's 11).
* a stored value: half a step of its group, plus what rounding scale and minimum to bf16 can
  move an end of the group: s / 2 + 15 * 2^-8 s + 2^-8 max|x|, plus the fp32 steps before.
* attention: rounding the probabilities, the values and the keys to bf16 (2^-8 each, where a
  kernel does) moves a score by at most d = 2^-8 scale sum|q k|, twice where q is rounded too,
  and so an output by (2 * 2^-8 + 4 d + 1e-4) sum p|v|; one rounding of the output; and over
  all outputs together, where such roundings average out, 1e-2 in the 2-norm.
"""

from __future__ import annotations

import math

import pytest
import torch

import kv4_reference as ref
from conftest import require_b200
from qtts_b200 import _native as nat
from qtts_b200 import kv4

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {"bf16": 2.0**-8, "fp16": 2.0**-11}


@pytest.fixture(autouse=True)
def _device():
    require_b200()
    nat.device_status(reset=True)
    yield
    torch.cuda.synchronize()
    assert nat.device_status(reset=True) == 0, "a kernel recorded a device-side failure"


def filled_cache(pages, kv_heads, page_size, d, g):
    cache = kv4.Kv4Cache.empty(pages, kv_heads, page_size, d)
    for name, keys in (("k", True), ("v", False)):
        x = torch.randn(pages, kv_heads, page_size, d, generator=g, dtype=torch.float64)
        codes, params = ref.write_rows(x, keys)
        getattr(cache, name + "_codes").copy_(codes)
        getattr(cache, name + "_params").copy_(params)
    return cache


def request_rows(cache, table_row, length):
    """Keys and values [length, Hkv, D] float64 of one request."""
    page = cache.page_size
    pages = table_row[: -(-length // page)].long()
    out = []
    for codes, params, keys in ((cache.k_codes, cache.k_params, True), (cache.v_codes, cache.v_params, False)):
        x = ref.read_rows(codes[pages], params[pages], keys)
        out.append(x.transpose(1, 2).reshape(-1, cache.kv_heads, cache.head_dim)[:length])
    return out


def check_attention(lengths, q_lens, heads, kv_heads, d, page, name, causal=True, seed=0, scale=None, ragged=None,
                    poison=False, q_gain=1.0):
    g = torch.Generator().manual_seed(seed)
    dtype, u = DTYPES[name], UNIT[name]
    batch = len(lengths)
    columns = max(1, max(-(-n // page) for n in lengths)) + 1
    pages = sum(-(-n // page) for n in lengths) + 2
    cache = filled_cache(pages, kv_heads, page, d, g)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.zeros(batch, columns, dtype=torch.int32)
    at, used = 0, []
    for b, n in enumerate(lengths):
        m = -(-n // page)
        table[b, :m] = order[at : at + m]
        used.append((order[at : at + m].tolist(), n))
        at += m
    if poison:  # everything that no request holds is NaN
        keep = torch.zeros(pages, page, dtype=torch.bool)
        for ids, n in used:
            for i, pid in enumerate(ids):
                keep[pid, : max(0, n - i * page)] = True
        for p in (cache.k_params, cache.v_params):
            p.masked_fill_(~keep.cuda()[:, None, :, None, None], float("nan"))
    total = sum(q_lens)
    q = (q_gain * torch.randn(total, heads, d, generator=g)).to(dtype).cuda()
    uniform = len(set(q_lens)) == 1 and not ragged
    starts = torch.tensor([sum(q_lens[:i]) for i in range(batch + 1)], dtype=torch.int32).cuda()
    table = table.cuda()
    out = kv4.kv4_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32).cuda(),
                            q_starts=None if uniform else starts, max_q=None if uniform else max(q_lens),
                            causal=causal, scale=scale)
    assert out.shape == q.shape and out.dtype == dtype
    sc = 1.0 / math.sqrt(d) if scale is None else scale
    err2 = ref2 = 0.0
    for b, (n, m) in enumerate(zip(lengths, q_lens)):
        k, v = request_rows(cache, table[b], n)
        i = torch.arange(m, device="cuda")
        sees = (n - m + i + 1).clamp_min(0) if causal else torch.full((m,), n, device="cuda")
        rows = slice(sum(q_lens[:b]), sum(q_lens[: b + 1]))
        want, mag, most = ref.attention(q[rows].double(), k, v, sees, sc)
        got = out[rows].double()
        assert torch.isfinite(got).all()
        d_score = 2.0**-8 * sc * most[..., None]
        bound = (2 * 2.0**-8 + 4 * d_score + 1e-4) * mag + u * want.abs() + 1e-7
        err = (got - want).abs()
        assert (err <= bound).all(), f"request {b}: {(err / bound).max().item():.2f} of the bound"
        err2 += err.square().sum().item()
        ref2 += want.square().sum().item()
    assert err2 <= (1e-2**2) * ref2 + 1e-12, f"2-norm {math.sqrt(err2 / ref2):.2e}"
    return out


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (8, 8), (5, 1), (32, 2), (20, 4)])
def test_single_tokens(name, d, heads, kv_heads):
    check_attention([1, 2, 15, 16, 17, 63, 64, 65, 200], [1] * 9, heads, kv_heads, d, 16, name)


@pytest.mark.parametrize("page", [16, 48, 64, 256, 768])
@pytest.mark.parametrize("length", [1, 47, 48, 129, 513, 1000])
def test_pages(page, length):
    check_attention([length, max(1, length - 13)], [1, 1], 16, 8, 128, page, "bf16", seed=page + length)


@pytest.mark.parametrize("length", [5000, 20011])
@pytest.mark.parametrize("batch", [1, 3])
def test_long_past(length, batch):
    check_attention([length - 7 * b for b in range(batch)], [1] * batch, 4, 2, 128, 64, "bf16", seed=length)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [2, 3, 5, 8, 17, 33])
@pytest.mark.parametrize("causal", [True, False])
def test_several_new_tokens(d, q_len, causal):
    check_attention([q_len, 40, 100], [q_len] * 3, 16, 8, d, 16, "bf16", causal=causal, seed=q_len)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (4, 4), (12, 2), (32, 4), (3, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(name, d, heads, kv_heads, causal):
    check_attention([130, 301, 257], [130, 301, 64], heads, kv_heads, d, 48, name, causal=causal, ragged=True)


@pytest.mark.parametrize("q_len,length", [(64, 64), (127, 127), (128, 128), (129, 129), (255, 1000), (256, 256),
                                          (512, 513), (700, 900)])
def test_prompt_edges(q_len, length):
    check_attention([length], [q_len], 4, 2, 128, 64, "bf16", seed=q_len)


@pytest.mark.parametrize("page,length", [(48, 912), (16, 890), (64, 1000), (64, 900)])
def test_prompts_over_tables_about_as_long_as_a_split(page, length):
    check_attention([length], [300], 4, 2, 128, page, "bf16", seed=length)


@pytest.mark.parametrize("rows", [63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("batch,length", [(1, 200), (3, 1500), (9, 1100)])
def test_rows_about_the_choice_of_kernel(rows, batch, length):
    check_attention([length - 5 * b for b in range(batch)], [rows] * batch, 4, 4, 64, 16, "fp16", seed=rows)


@pytest.mark.parametrize("k_lift,v_lift", [(0, 0), (60, -40), (-30, 90)])
@pytest.mark.parametrize("q_len", [1, 300])
def test_bf16_beyond_the_range_of_fp16(q_len, k_lift, v_lift):
    # Keys and values far outside fp16's range, values that differ by 2^24 from page to page and a page
    # of zeros, against the formula with the bound of check_attention.
    g = torch.Generator().manual_seed(9)
    cache = filled_cache(40, 2, 16, 128, g)
    by_page = 2.0 ** torch.randint(-12, 13, (40, 1, 1, 1, 1), generator=g).cuda()
    by_page[7] = 0.0
    cache.k_params.copy_(cache.k_params.float() * 2.0**k_lift)
    cache.v_params.copy_(cache.v_params.float() * by_page * 2.0**v_lift)
    q = torch.randn(q_len, 4, 128, generator=g).to(torch.bfloat16).cuda()
    table = torch.arange(40, dtype=torch.int32).cuda()[None]
    n, sc = 633, 128**-0.5 * 2.0**-k_lift
    out = kv4.kv4_attention(q, cache, table, torch.tensor([n], dtype=torch.int32).cuda(), scale=sc).double()
    k, v = request_rows(cache, table[0], n)
    sees = n - q_len + torch.arange(q_len, device="cuda") + 1
    want, mag, most = ref.attention(q.double(), k, v, sees, sc)
    bound = (2 * 2.0**-8 + 4 * 2.0**-8 * sc * most[..., None] + 1e-4) * mag + UNIT["bf16"] * want.abs()
    assert ((out - want).abs() <= bound).all()


def test_ragged_chunks_with_empty_requests():
    check_attention([70, 0, 300, 9], [70, 0, 129, 1], 16, 8, 128, 16, "bf16", ragged=True)


def test_rows_that_see_nothing_are_zeros():
    # Five new tokens in a request that holds three: the first two see nothing; an empty request.
    out = check_attention([3, 0, 4], [5, 5, 5], 4, 2, 128, 16, "bf16")
    assert (out[:2] == 0).all() and (out[5:10] == 0).all() and (out[10] == 0).all() and (out[2] != 0).any()
    out = check_attention([40, 0], [100, 100], 4, 2, 128, 16, "bf16")
    assert (out[:60] == 0).all() and (out[100:] == 0).all()


@pytest.mark.parametrize("q_len", [1, 4, 40, 200])
@pytest.mark.parametrize("page", [16, 64])
def test_nothing_outside_a_request_is_used(q_len, page):
    check_attention([q_len + 3, 211, 260], [q_len] * 3, 8, 4, 128, page, "bf16", poison=True, seed=q_len)


@pytest.mark.parametrize("q_len", [4, 150])
def test_nan_in_tokens_that_a_row_does_not_see(q_len):
    g = torch.Generator().manual_seed(5)
    cache = filled_cache(8, 2, 64, 128, g)
    q = torch.randn(q_len, 4, 128, generator=g).to(torch.bfloat16).cuda()
    table = torch.arange(8, dtype=torch.int32).cuda()[None]
    lengths = torch.tensor([q_len + 30], dtype=torch.int32).cuda()
    clean = kv4.kv4_attention(q, cache, table, lengths)
    last = q_len + 29
    for p in (cache.k_params, cache.v_params):
        p[last // 64, :, last % 64] = float("nan")
    dirty = kv4.kv4_attention(q, cache, table, lengths)
    assert torch.equal(clean[:-1], dirty[:-1]) and torch.isnan(dirty[-1].float()).all()


@pytest.mark.parametrize("q_len", [1, 130])
def test_sharp_scores(q_len):
    # Scores of some hundreds: the running maximum moves, most probabilities are zero.
    check_attention([400], [q_len], 8, 4, 128, 16, "bf16", scale=0.5, q_gain=4.0, seed=11)


@pytest.mark.parametrize("q_len", [1, 3, 70])
def test_strided_q_and_table(q_len):
    g = torch.Generator().manual_seed(3)
    cache = filled_cache(12, 4, 16, 128, g)
    fused = torch.randn(2 * q_len, 16, 128, generator=g).to(torch.bfloat16).cuda()
    q = fused[:, 3:11]  # heads inside a fused projection's rows
    wide = torch.randperm(12, generator=g).to(torch.int32).reshape(2, 6).cuda()
    lengths = torch.tensor([75, 71], dtype=torch.int32).cuda()
    a = kv4.kv4_attention(q, cache, wide[:, :5], lengths)
    b = kv4.kv4_attention(q.contiguous(), cache, wide[:, :5].contiguous(), lengths)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)  # 2-byte aligned
    odd.copy_(q)
    c = kv4.kv4_attention(odd, cache, wide[:, :5], lengths)
    assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("q_len", [1, 100])
def test_same_bits_again_and_on_another_stream(q_len):
    g = torch.Generator().manual_seed(4)
    cache = filled_cache(40, 2, 64, 128, g)
    q = torch.randn(2 * q_len, 4, 128, generator=g).to(torch.bfloat16).cuda()
    table = torch.arange(40, dtype=torch.int32).cuda().view(2, 20)
    lengths = torch.tensor([1280, 900], dtype=torch.int32).cuda()
    first = kv4.kv4_attention(q, cache, table, lengths)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        others = [kv4.kv4_attention(q, cache, table, lengths) for _ in range(5)]
    side.synchronize()
    for o in others:
        assert torch.equal(first, o)


def test_out_of_range_indices_are_recorded():
    g = torch.Generator().manual_seed(6)
    cache = filled_cache(4, 2, 16, 128, g)
    q = torch.randn(1, 4, 128, generator=g).to(torch.bfloat16).cuda()
    good = torch.tensor([[1, 2, 3]], dtype=torch.int32).cuda()
    kv4.kv4_attention(q, cache, torch.tensor([[1, 9, -1]], dtype=torch.int32).cuda(),
                      torch.tensor([40], dtype=torch.int32).cuda())
    assert nat.device_status(reset=True) == 2
    kv4.kv4_attention(q, cache, good, torch.tensor([49], dtype=torch.int32).cuda())
    assert nat.device_status(reset=True) == 2
    # A request of more new tokens than max_q says.
    q3 = torch.randn(3, 4, 128, generator=g).to(torch.bfloat16).cuda()
    kv4.kv4_attention(q3, cache, good, torch.tensor([20], dtype=torch.int32).cuda(),
                      q_starts=torch.tensor([0, 3], dtype=torch.int32).cuda(), max_q=2)
    assert nat.device_status(reset=True) == 2


# ---- the writer ---------------------------------------------------------------------------------


def tables(length, d, theta=1.0e6):
    ang = torch.arange(length, dtype=torch.float32)[:, None] / theta ** (torch.arange(0, d, 2).float() / d)
    return torch.cos(ang).cuda(), torch.sin(ang).cuda()


def axis_of(j, sections, interleaved):
    if interleaved:
        a = j % len(sections)
        return a if j < len(sections) * sections[a] else 0
    for a, n in enumerate(sections):
        if j < n:
            return a
        j -= n
    raise AssertionError


def expected_rows(x, weight, eps, cos, sin, positions, sections, interleaved):
    """x [T, H, D] float64 through the norm and the rotation."""
    if weight is not None:
        x = weight.double() * x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if cos is None:
        return x
    half = x.shape[-1] // 2
    y = x.clone()
    for j in range(half):
        pos = positions[axis_of(j, sections, interleaved)]
        c, s = cos[pos, j].double()[:, None], sin[pos, j].double()[:, None]
        y[..., j] = x[..., j] * c - x[..., j + half] * s
        y[..., j + half] = x[..., j + half] * c + x[..., j] * s
    return y


def check_write(tokens, heads, kv_heads, d, page, name, axes=1, sections=None, interleaved=False, norm=True, rope=True,
                seed=0, skip=(), gain=1.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    dtype, u = DTYPES[name], UNIT[name]
    pages = -(-tokens // page) + 2
    cache = filled_cache(pages, kv_heads, page, d, g)
    before = [t.clone() for t in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params)]
    width = (heads + 2 * kv_heads) * d
    qkv = (gain * torch.randn(tokens, width + pad, generator=g)).to(dtype).cuda()[:, :width]
    slots = torch.randperm(pages * page, generator=g)[:tokens].cuda()
    for i in skip:
        slots[i] = -1
    cos, sin = tables(300, d) if rope else (None, None)
    positions = torch.randint(0, 300, (axes, tokens), generator=g).cuda() if rope else None
    sections = sections or (d // 2,)
    qw = (1 + 0.2 * torch.randn(d, generator=g)).to(dtype).cuda() if norm else None
    kw = (1 + 0.2 * torch.randn(d, generator=g)).to(dtype).cuda() if norm else None
    q, k_held, v_held = kv4.rope_kv4_append(
        qkv, cache, slots, heads, cos=cos, sin=sin, positions=positions, sections=sections if rope else None,
        interleaved=interleaved, q_norm=qw, k_norm=kw, eps=1e-6, values=True)
    x = qkv.double().reshape(tokens, heads + 2 * kv_heads, d)
    args = (1e-6, cos, sin, positions, sections, interleaved)
    want_q = expected_rows(x[:, :heads], qw, *args)
    top = want_q.abs().amax(-1, keepdim=True) if heads else want_q
    assert q.shape == (tokens, heads, d)
    assert ((q.double() - want_q).abs() <= u * want_q.abs() + 1e-5 * top + 2.0**-24).all()
    stored = (slots >= 0).nonzero().flatten()
    which, row = slots[stored] // page, slots[stored] % page
    for want, held, codes, params, keys in (
            (expected_rows(x[:, heads : heads + kv_heads], kw, *args), k_held, cache.k_codes, cache.k_params, True),
            (x[:, heads + kv_heads :], v_held, cache.v_codes, cache.v_params, False)):
        got = ref.read_rows(codes[which, :, row], params[which, :, row], keys)
        s = params[which, :, row][..., 0].double().repeat_interleave(32, -1)
        w = want[stored]
        top = w.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
        row_top = w.abs().amax(-1, keepdim=True)
        assert ((got - w).abs() <= s * (0.5 + 15 * 2.0**-8) + 2.0**-8 * top + 1e-5 * row_top).all()
        # The values handed out are the cache's, rounded once (fp32 on the way).
        assert ((held[stored].double() - got).abs() <= u * got.abs() + 1e-6 * top + 2.0**-24).all()
    # Nothing else was touched.
    keep = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    keep[which, row] = False
    for now, then in zip((cache.k_codes, cache.k_params, cache.v_codes, cache.v_params), before):
        a, b = now.transpose(1, 2)[keep], then.transpose(1, 2)[keep]
        assert torch.equal(a, b)
    k_read, v_read = cache.values()
    assert torch.equal(k_read.double(), ref.read_rows(cache.k_codes, cache.k_params, True).float().double())
    assert torch.equal(v_read.double(), ref.read_rows(cache.v_codes, cache.v_params, False).float().double())
    alone = kv4.rope_kv4_append(qkv, cache, slots, heads, cos=cos, sin=sin, positions=positions,
                                sections=sections if rope else None, interleaved=interleaved, q_norm=qw, k_norm=kw)
    assert torch.equal(alone, q)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 7, 65])
def test_write(name, d, tokens):
    check_write(tokens, 16, 8, d, 16, name, seed=tokens)


@pytest.mark.parametrize("d,sections", [(64, (16, 8, 8)), (128, (24, 20, 20)), (128, (64, 0, 0)), (128, (0, 1, 63)),
                                        (64, (8, 8, 8, 8)), (128, (30, 34))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_write_with_axes(d, sections, interleaved):
    check_write(33, 6, 3, d, 48, "bf16", axes=len(sections), sections=sections, interleaved=interleaved)


@pytest.mark.parametrize("norm,rope", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("heads,kv_heads", [(0, 2), (1, 1), (20, 4), (3, 3)])
def test_write_parts(norm, rope, heads, kv_heads):
    check_write(19, heads, kv_heads, 128, 16, "bf16", norm=norm, rope=rope)


def test_write_skips_strides_and_sizes():
    check_write(50, 16, 8, 128, 64, "bf16", skip=(0, 7, 49))
    check_write(50, 16, 8, 64, 64, "fp16", pad=24)
    check_write(9, 4, 2, 128, 16, "bf16", pad=5)  # rows that are not 16-byte aligned
    check_write(21, 4, 2, 128, 16, "bf16", gain=1e4, norm=False)
    check_write(21, 4, 2, 128, 16, "bf16", gain=1e-6, norm=False)


def test_write_constant_and_non_finite_groups():
    cache = kv4.Kv4Cache.empty(1, 1, 16, 64)
    qkv = torch.zeros(5, 2 * 64, dtype=torch.bfloat16, device="cuda")
    qkv[1] = 3.0
    qkv[2] = torch.randn(128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    qkv[3], qkv[4] = qkv[2], qkv[2]
    qkv[2, 5] = float("inf")
    qkv[3, 5] = float("nan")
    qkv[4, 69] = float("-inf")
    kv4.rope_kv4_append(qkv, cache, torch.arange(5).cuda(), 0)
    k, v = (t[0, 0] for t in cache.values())
    assert (k[0] == 0).all() and (v[0] == 0).all() and (k[1] == 3).all() and (v[1] == 3).all()
    for i in (2, 3):
        assert not torch.isfinite(k[i, :32]).any() and torch.isfinite(k[i, 32:]).all() and torch.isfinite(v[i]).all()
    assert not torch.isfinite(v[4, :32]).any() and torch.isfinite(v[4, 32:]).all() and torch.isfinite(k[4]).all()


def test_write_out_of_range_is_recorded_and_not_stored():
    cache = kv4.Kv4Cache.empty(2, 1, 16, 64)
    qkv = torch.randn(3, 3 * 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()
    cos, sin = tables(10, 64)
    kv4.rope_kv4_append(qkv, cache, torch.tensor([0, 32, 1]).cuda(), 1)
    assert nat.device_status(reset=True) == 2
    assert (cache.k_params[0, 0, :2] != 0).any() and (cache.k_params[1] == 0).all()
    cache = kv4.Kv4Cache.empty(2, 1, 16, 64)
    q = kv4.rope_kv4_append(qkv, cache, torch.tensor([0, 1, 2]).cuda(), 1, cos=cos, sin=sin,
                            positions=torch.tensor([3, 10, -1]).cuda())
    assert nat.device_status(reset=True) == 2
    assert (q[0] != 0).any() and (q[1:] == 0).all()
    assert (cache.v_params[0, 0, 0] != 0).any() and (cache.v_params[0, 0, 1:] == 0).all()


def test_write_then_attend_in_a_graph():
    g = torch.Generator().manual_seed(9)
    cache = filled_cache(4, 8, 64, 128, g)
    qkv = torch.randn(2, 32 * 128, generator=g).to(torch.bfloat16).cuda()
    cos, sin = tables(200, 128)
    positions = torch.tensor([100, 60]).cuda()
    slots = torch.tensor([64 + 36, 192 + 2]).cuda()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    lengths = torch.tensor([101, 67], dtype=torch.int32).cuda()

    def step():
        q = kv4.rope_kv4_append(qkv, cache, slots, 16, cos=cos, sin=sin, positions=positions)
        return kv4.kv4_attention(q, cache, table, lengths)

    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    qkv2 = torch.randn(2, 32 * 128, generator=g).to(torch.bfloat16).cuda()
    saved = qkv.clone()
    qkv.copy_(qkv2)
    graph.replay()
    assert not torch.equal(got, want)
    qkv.copy_(saved)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
