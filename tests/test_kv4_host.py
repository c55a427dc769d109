"""Refusals of the 4-bit cache, its attention and the fused residual norm: on the host, before
any launch, so no GPU is needed to see them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from qtts_b200 import _native as nat
from qtts_b200 import kv4
from qtts_b200.quant import kernels as qk

OK, NULL, SHAPE, ALIGN, DTYPE, ARCH = 0, 1, 2, 3, 4, 5


@pytest.fixture(scope="module")
def lib():
    return nat.lib()


def valid_answer():
    return ARCH if not torch.cuda.is_available() else None


def norm_quant(lib, x=16, ldx=64, r=16, ldr=64, w=16, ro=16, ldro=64, dtype=nat.BF16, q=16, ldq=64, to=nat.E4M3,
               scale=16, rows=4, width=64):
    return lib.qtts_add_rms_norm_quant(x, ldx, r, ldr, w, 1e-6, ro, ldro, dtype, q, ldq, to, scale, rows, width, 0,
                                       None)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(rows=-1)), (SHAPE, dict(width=0)), (SHAPE, dict(width=65537, ldx=1 << 17)), (OK, dict(rows=0, x=None)),
    (NULL, dict(x=None)), (NULL, dict(w=None)), (NULL, dict(q=None)), (NULL, dict(scale=None)), (NULL, dict(r=None)),
    (NULL, dict(ro=None)), (DTYPE, dict(dtype=nat.INT8)), (DTYPE, dict(to=nat.BF16)), (SHAPE, dict(ldx=63)),
    (SHAPE, dict(ldr=63)), (SHAPE, dict(ldro=63)), (SHAPE, dict(ldq=63)), (ALIGN, dict(x=17)), (ALIGN, dict(scale=18)),
    (ALIGN, dict(ro=18, dtype=nat.FP32)),
])
def test_norm_quant_refuses(lib, want, kw):
    assert norm_quant(lib, **kw) == want


def write(lib, qkv=16, ldqkv=32 * 128, dtype=nat.BF16, tokens=3, heads=16, kv_heads=8, d=128, qn=None, kn=None, cos=16,
          sin=16, length=10, pos=16, ldpos=3, sections=(64,), axes=None, interleaved=0, slots=16, q=16, ldq=16 * 128,
          kc=16, kp=16, vc=16, vp=16, pages=2, page=16, kval=None, vval=None):
    arr = (ctypes.c_int * max(1, len(sections)))(*sections) if sections is not None else None
    return lib.qtts_rope_kv4_append(qkv, ldqkv, dtype, tokens, heads, kv_heads, d, qn, kn, 1e-6, cos, sin, length, pos,
                                    ldpos, len(sections) if axes is None else axes, arr, interleaved, slots, q, ldq, kc,
                                    kp, vc, vp, pages, page, kval, vval, 0, None)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(tokens=-1)), (SHAPE, dict(kv_heads=0)), (SHAPE, dict(heads=-1)), (SHAPE, dict(d=96)),
    (SHAPE, dict(pages=-1)), (SHAPE, dict(page=0)), (DTYPE, dict(dtype=nat.FP32)), (OK, dict(tokens=0, qkv=None)),
    (NULL, dict(qkv=None)), (NULL, dict(slots=None)), (NULL, dict(q=None)), (NULL, dict(kc=None)), (NULL, dict(vp=None)),
    (NULL, dict(cos=None)), (NULL, dict(pos=None)), (NULL, dict(sections=None, axes=1)), (NULL, dict(kval=16)),
    (SHAPE, dict(ldqkv=32 * 128 - 8)), (SHAPE, dict(ldq=15 * 128)), (SHAPE, dict(sections=(63,))),
    (SHAPE, dict(sections=(65, -1))), (SHAPE, dict(sections=(16, 16, 16, 8, 8))), (SHAPE, dict(length=0)),
    (SHAPE, dict(ldpos=2)), (ALIGN, dict(qkv=24)), (ALIGN, dict(ldqkv=32 * 128 + 4)), (ALIGN, dict(q=20)),
    (ALIGN, dict(qn=2)), (ALIGN, dict(slots=4)), (ALIGN, dict(kp=4)), (ALIGN, dict(kval=8, vval=16)),
])
def test_write_refuses(lib, want, kw):
    assert write(lib, **kw) == want


def attend(lib, q=16, qt=16 * 128, qh=128, dtype=nat.BF16, kc=16, kp=16, vc=16, vp=16, pages=4, page=16, table=16,
           ld=2, cols=2, lengths=16, starts=None, total=3, max_q=1, batch=3, heads=16, kv_heads=8, d=128, out=16,
           ot=16 * 128, scale=0.1, workspace=None):
    return lib.qtts_kv4_attention(q, qt, qh, dtype, kc, kp, vc, vp, pages, page, table, ld, cols, lengths, starts, total,
                                  max_q, batch, heads, kv_heads, d, scale, 1, out, ot, workspace, 0, None)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(batch=-1)), (SHAPE, dict(batch=65536, total=65536)), (SHAPE, dict(total=-1)), (SHAPE, dict(max_q=4)),
    (SHAPE, dict(heads=12)), (SHAPE, dict(kv_heads=0)), (SHAPE, dict(d=80)), (SHAPE, dict(page=24)), (SHAPE, dict(page=8)),
    (SHAPE, dict(cols=3)), (SHAPE, dict(cols=-1)), (DTYPE, dict(dtype=nat.FP32)), (OK, dict(batch=0, total=0, max_q=0)),
    (OK, dict(total=0, max_q=0, q=None)), (SHAPE, dict(total=4)), (SHAPE, dict(cols=1 << 27, ld=1 << 27, page=16)),
    (NULL, dict(q=None)), (NULL, dict(out=None)), (NULL, dict(lengths=None)), (NULL, dict(table=None)),
    (NULL, dict(kc=None)), (NULL, dict(vp=None)), (SHAPE, dict(qh=64)), (SHAPE, dict(ot=15 * 128)), (ALIGN, dict(q=24)),
    (ALIGN, dict(qt=16 * 128 + 4)), (ALIGN, dict(out=8)), (ALIGN, dict(table=2)), (ALIGN, dict(starts=2)),
    (ALIGN, dict(vc=8)), (SHAPE, dict(scale=0.0)), (SHAPE, dict(scale=-1.0)), (SHAPE, dict(scale=float("nan"))),
    (SHAPE, dict(scale=float("inf"))),
])
def test_attention_refuses(lib, want, kw):
    assert attend(lib, **kw) == want


def test_valid_arguments_reach_the_device_check(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert norm_quant(lib) == norm_quant(lib, r=None, ro=None) == ARCH
    assert write(lib) == write(lib, cos=None, sin=None) == write(lib, sections=(24, 20, 20)) == ARCH
    assert write(lib, heads=0, q=None) == ARCH
    assert attend(lib) == attend(lib, starts=16, total=7, max_q=5) == ARCH


def test_workspace(lib):
    def need(total=1, max_q=1, batch=1, heads=16, kv_heads=8, d=128, tokens=64):
        return lib.qtts_kv4_attention_workspace(total, max_q, batch, heads, kv_heads, d, tokens)

    assert need() == need(total=0) == need(batch=0) == need(heads=12) == 0
    assert need(total=64, batch=64, tokens=1 << 20) == 0  # many requests: no split across the workspace
    long = need(tokens=1 << 20)
    assert long > 0 and long % (16 * (128 + 2) * 4) == 0
    kw = dict(total=1, batch=1, cols=1 << 16, ld=1 << 16)
    assert attend(lib, **kw) == NULL and attend(lib, workspace=8, **kw) == ALIGN


def cache(**kw):
    a = dict(pages=2, kv_heads=2, page_size=16, head_dim=64) | kw
    return kv4.Kv4Cache.empty(a["pages"], a["kv_heads"], a["page_size"], a["head_dim"], device="cpu")


def test_cache_refuses():
    c = cache()
    assert c.nbytes == 2 * 2 * 2 * 16 * (32 + 8)
    for kw in (dict(head_dim=96), dict(page_size=24), dict(page_size=0)):
        with pytest.raises(ValueError):
            cache(**kw)
    with pytest.raises(ValueError):
        kv4.Kv4Cache(c.k_codes, c.k_params.float(), c.v_codes, c.v_params)
    with pytest.raises(ValueError):
        kv4.Kv4Cache(c.k_codes, c.k_params[:1], c.v_codes, c.v_params)
    with pytest.raises(ValueError):
        kv4.Kv4Cache(c.k_codes.int(), c.k_params, c.v_codes, c.v_params)
    with pytest.raises(ValueError):
        kv4.Kv4Cache(c.k_codes.transpose(0, 1), c.k_params, c.v_codes, c.v_params)


def test_wrappers_refuse():
    c = cache()
    qkv, slots = torch.zeros(3, 8 * 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    table, pos = torch.zeros(10, 32), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv4.rope_kv4_append(qkv, c, slots, 4)
    for kw, err in ((dict(qkv=qkv[:, :-8]), ValueError), (dict(qkv=qkv.float()), TypeError),
                    (dict(slots=slots.int()), ValueError), (dict(slots=slots[:2]), ValueError),
                    (dict(cos=table), ValueError)):
        a = dict(qkv=qkv, slots=slots) | kw
        with pytest.raises(err):
            kv4.rope_kv4_append(a.pop("qkv"), c, a.pop("slots"), 4, **a)
    q, bt, ln = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32), torch.ones(
        2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv4.kv4_attention(q, c, bt, ln)
    for args, kw, err in (((q[:, :3], c, bt, ln), {}, ValueError), ((q.float(), c, bt, ln), {}, TypeError),
                          ((q, c, bt.long(), ln), {}, ValueError), ((q, c, bt, ln.long()), {}, ValueError),
                          ((q, c, bt[:1], ln), {}, ValueError), ((q[:1], c, bt, ln), {}, ValueError),
                          ((q, c, bt, ln), dict(q_starts=torch.zeros(3, dtype=torch.int32)), ValueError),
                          ((q, c, bt, ln), dict(q_starts=torch.zeros(2, dtype=torch.int32), max_q=1), ValueError)):
        with pytest.raises(err):
            kv4.kv4_attention(*args, **kw)
    x, w = torch.zeros(2, 64), torch.ones(64)
    with pytest.raises(RuntimeError, match="CUDA"):
        qk.add_rms_norm_quant(x, x, w)
    for args, kw, err in (((x, x, w[:32]), {}, ValueError), ((x, x, w), dict(dtype=torch.uint8), TypeError)):
        with pytest.raises(err):
            qk.add_rms_norm_quant(*args, **kw)


def test_fast_calls_convert_as_ctypes_does(lib):
    """The converted-argument calls against ctypes: the same answers, and errors instead of
    wrong conversions."""
    fast = nat._fastcall()
    if fast is None:
        pytest.skip("csrc/fastcall.c is not built here")

    def both(name, args):
        slow = nat._through_ctypes(name)
        assert getattr(fast, name)(*args) == slow(*args)

    norm = [16, 64, 16, 64, 16, 1e-6, 16, 64, nat.BF16, 16, 64, nat.E4M3, 16, 4, 64, 0, None]
    write_args = [16, 32 * 128, nat.BF16, 3, 16, 8, 128, None, None, 1e-6, 16, 16, 10, 16, 3, 1, (64,), False, 16, 16,
                  16 * 128, 16, 16, 16, 16, 2, 16, None, None, 0, None]
    attend_args = [16, 16 * 128, 128, nat.BF16, 16, 16, 16, 16, 4, 16, 16, 2, 2, 16, None, 3, 1, 3, 16, 8, 128, 0.1, True,
                   16, 16 * 128, None, 0, None]
    for name, args, bad in (("qtts_add_rms_norm_quant", norm, (13, 14, 1, 8, 11)),
                            ("qtts_rope_kv4_append", write_args, (3, 5, 1, 2, 26)),
                            ("qtts_kv4_attention", attend_args, (17, 19, 1, 3, 9))):
        if not torch.cuda.is_available():
            both(name, args)
        for at in bad:
            both(name, args[:at] + [-1] + args[at + 1:])
        both(name, [None] + args[1:])
        both(name, [1 << 40 | 1] + args[1:])
        with pytest.raises(TypeError):
            getattr(fast, name)(*args[:-1])
        with pytest.raises(TypeError):
            getattr(fast, name)("x", *args[1:])
        with pytest.raises(OverflowError):
            getattr(fast, name)(*args[:3], *[1 << 40 if i == bad[0] else a for i, a in enumerate(args) if i >= 3])
    for sections in ((24, 20, 20), (63,), None):
        both("qtts_rope_kv4_append", write_args[:15] + [len(sections or (1,)), sections] + write_args[17:])
    with pytest.raises(TypeError):
        fast.qtts_rope_kv4_append(*write_args[:16], (1, 2, 3, 4, 5), *write_args[17:])
    with pytest.raises(TypeError):
        fast.bind(1, 2)


def test_no_workspace_below_the_split():
    # The Python entry does not ask for a workspace below this many tokens, so none may be needed.
    for heads, kv_heads in [(1, 1), (16, 8), (32, 4), (5, 1)]:
        for max_q in (1, 3, 20, 64, 300, 2000):
            for batch in (1, 2, 9, 64):
                for d in (64, 128):
                    args = (batch * max_q, max_q, batch, heads, kv_heads, d)
                    for tokens in (16, 500, kv4._SPLIT_FROM - 1):
                        assert nat.lib().qtts_kv4_attention_workspace(*args, tokens) == 0
    assert nat.lib().qtts_kv4_attention_workspace(300, 300, 1, 4, 2, 128, kv4._SPLIT_FROM) > 0
