"""The talker's decode step over the 4-bit cache: the fused path against the same step in torch ops
on the values that the cache holds, alone and with W8A8 projections, and a captured frame.

Bars: in the unquantized model every op rounds to bf16 on both sides (2^-8 a value at most), some ten
roundings a layer that do not share an order: 3e-2 of the hidden state in the 2-norm over two layers.
W8A8 adds the e4m3 or int8 codes of activations that differ by such roundings: where a code
flips it moves by a step (2^-3 of a value for e4m3): 6e-2.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from conftest import require_b200
from qtts_b200 import _native as nat
from qtts_b200.decode_step import Frame, Talker, apply_rope, random_init_, rms_norm
from qtts_b200.quant.fp8 import Fp8Method
from qtts_b200.quant.int8 import Int8Method
from qtts_b200.layers.linear import iter_linears

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    require_b200()
    nat.device_status(reset=True)
    yield
    torch.cuda.synchronize()
    assert nat.device_status() == 0


def plain_step(talker: Talker, x: torch.Tensor) -> torch.Tensor:
    """Talker.step's hidden state by torch ops, keys and values as the 4-bit caches give them."""
    b, d = x.shape[0], talker.d
    h = x[:, None, :]
    for layer, cache in zip(talker.layers, talker.kv4):
        q, k, v = layer._qkv(h, talker.cos, talker.sin)
        keys, values = cache.values()  # [streams, kv_heads, slots, head_dim]; the new token is in it
        n = talker.pos + 1
        att = F.scaled_dot_product_attention(q.float(), keys[:, :, :n], values[:, :, :n], enable_gqa=True)
        h = h + layer.o_proj(att.to(h.dtype).transpose(1, 2).reshape(b, 1, -1))
        h = layer._mlp(h)
    return rms_norm(h[:, 0], talker.norm)


@pytest.mark.parametrize("method,bar", [(None, 3e-2), (Fp8Method, 6e-2), (Int8Method, 6e-2)])
@pytest.mark.parametrize("batch", [1, 5])
def test_step_against_torch_ops(method, bar, batch):
    talker = Talker(batch, layers=2, seed=3, kv_cache="int4")
    random_init_(talker, 0)
    if method is not None:
        m = method()
        for name, linear in iter_linears(talker):
            if "head" not in name:
                m.process_weights(linear)
                linear.quant_method = m
    x = torch.randn(batch, talker.d.hidden, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    with torch.no_grad():
        hidden, codes = talker.step(x)
        want = plain_step(talker, x)
    err = (hidden.float() - want.float()).norm() / want.float().norm()
    assert err <= bar, f"{err:.3e}"
    assert codes.shape == (batch,) and ((codes >= 1) & (codes < 2048) | (codes == 2150)).all()


def test_four_bits_stay_near_sixteen():
    # The same streams over both caches: 4-bit keys and values of N(0, 1) are off by some 8 % each
    # (a step of 4.1 sigma / 15, uniform error), which 512 tokens average out.
    x = torch.randn(3, 2048, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    hidden = []
    for kind in ("bf16", "int4"):
        talker = Talker(3, layers=2, seed=3, kv_cache=kind)
        random_init_(talker, 0)
        with torch.no_grad():
            hidden.append(talker.step(x)[0].float())
    assert (hidden[0] - hidden[1]).norm() <= 0.1 * hidden[0].norm()


def test_frame_in_a_graph_with_a_4_bit_cache():
    frame = Frame(4, talker_layers=2, predictor_layers=1, codebooks=2, kv_cache="int4")
    m = Fp8Method()
    for name, linear in iter_linears(frame.talker):
        if "head" not in name:
            m.process_weights(linear)
            linear.quant_method = m
    with torch.no_grad():
        want = frame.run().clone()
    frame.capture()
    frame.codes.zero_()
    frame.graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(frame.codes, want)


def test_unknown_cache_is_refused():
    with pytest.raises(ValueError, match="kv_cache"):
        Talker(1, layers=1, kv_cache="int2")
