"""Prefill in key splits over values far from 1: the splits' fp16 states carry a row exponent in both directions, so a power
of two on V comes out of the call as that power of two on the result, and infinities in one channel leave the others'."""

import numpy as np
import pytest
import torch

from cases import as_np32
from engine.hip_decode import QuantKV
from engine.hip_prefill import paged_prefill_attention
from oracle import paged_ref
from test_prefill_gpu import SHAPES, assert_bf16_close, make_prefill

pytestmark = pytest.mark.gpu
CTX, QLEN = [1500, 700], [70, 33]


@pytest.mark.parametrize("shape", ["0.5B", "1.5B", "g3"])
@pytest.mark.parametrize("layout", ["auto", "w8x1", "w16x1", "w16h2"])
@pytest.mark.parametrize("int8", [False, True])
def test_a_power_of_two_on_v_is_one_on_the_result(shape, layout, int8):
    """Every fp32 sum, fp16 state and bf16 result scales by 2^e exactly: equal bits. (V at 2^e, |V| about 2^-12 to 4 times it.)"""
    Hq, Hkv, D = SHAPES[shape]
    q, k, v, bt, c, st, ln = make_prefill(CTX, QLEN, Hq, Hkv, D, seed=81)[:7]
    one = torch.full(v.shape[:3], 1 / 64, device="cuda")
    kq, vq = ((t.float() * 64).round().clamp(-127, 127).to(torch.int8) for t in (k, v))

    def run(e, splits):
        print(f"case prefill V 2^{e} shape={shape} layout={layout} int8={int8} splits={splits}", flush=True)
        kv = (kq, vq) if int8 else (k, v * 2.0 ** e)
        quant = QuantKV(1, one, one * 2.0 ** e) if int8 else None
        return paged_prefill_attention(q, *kv, bt, c, st, ln, D ** -0.5, max(CTX), max(QLEN), num_splits=splits, wg_layout=layout,
                                       quant=quant).double()

    for splits in (1, 2, 6):
        base = run(0, splits)
        for e in (-90, -40, -30, -24, -20, -16, -14, -4, 14, 15, 30, 90):
            assert torch.equal(run(e, splits) * 2.0 ** -e, base), f"2^{e}, {splits} splits"


@pytest.mark.parametrize("shape", ["0.5B", "1.5B"])
@pytest.mark.parametrize("splits", [1, 2, 6])
def test_an_infinite_channel_beside_large_finite_ones(shape, splits):
    Hq, Hkv, D = SHAPES[shape]
    q, k, v, bt, c, st, ln, tables, starts, T = make_prefill(CTX, QLEN, Hq, Hkv, D, seed=82)
    print(f"case prefill infinite channel shape={shape} splits={splits}", flush=True)
    bad = v * 2.0 ** 20
    bad[:, tables[0][3], 5, 7] = float("inf")
    out = paged_prefill_attention(q, k, bad, bt, c, st, ln, D ** -0.5, max(CTX), max(QLEN), num_splits=splits)
    ref = paged_ref.prefill(as_np32(q), as_np32(k), as_np32(v), tables, CTX, starts, QLEN, D ** -0.5, dtype=np.float32)
    assert (out[:QLEN[0], :, 7] == float("inf")).all()
    out[:QLEN[0], :, 7] = 0
    ref[:QLEN[0], :, 7] = 0
    assert_bf16_close(out.double().cpu().numpy() / 2.0 ** 20, ref, "beside an infinite channel")


@pytest.mark.parametrize("shape", ["0.5B", "1.5B"])
def test_rows_of_small_and_large_channels(shape):
    """Channels from 2^-12 to 2^12 side by side keep their own precision: fp16 holds 2^29 below a row's largest in full."""
    Hq, Hkv, D = SHAPES[shape]
    q, k, v, bt, c, st, ln, tables, starts, T = make_prefill(CTX, QLEN, Hq, Hkv, D, seed=83)
    print(f"case prefill channels shape={shape}", flush=True)
    by = torch.exp2(torch.linspace(-12, 12, D, device="cuda").round())
    out = paged_prefill_attention(q, k, v * by.bfloat16(), bt, c, st, ln, D ** -0.5, max(CTX), max(QLEN), num_splits=5)
    ref = paged_ref.prefill(as_np32(q), as_np32(k), as_np32(v), tables, CTX, starts, QLEN, D ** -0.5, dtype=np.float32)
    assert_bf16_close((out.double() / by.double()).cpu().numpy(), ref, "channels of their own magnitudes")
