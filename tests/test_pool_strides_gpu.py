"""Pools whose layers are contiguous although a dimension of one entry has another stride: every plan takes them, as the decode's."""

import pytest
import torch

from engine.hip_decode import DecodePlan
from engine.hip_prefix import PrefixPlan
from engine.hip_tree import TreePlan
from prefix_cases import batch, check
from tree_cases import Case

pytestmark = pytest.mark.gpu


def odd(pool):
    """Two layers [2, 1, N, B, D] of one KV head whose dimension lies where no contiguous pool has it."""
    _, N, B, D = pool.shape
    t = torch.zeros(2, N, 1, B, D, dtype=pool.dtype, device="cuda").transpose(1, 2)
    t[1] = pool
    assert t[1].is_contiguous() and t.stride()[1] != pool.numel() and torch.equal(t[1].view(torch.int16), pool.view(torch.int16))
    return t


def test_layers_of_one_head():
    x = batch([(128, [20, 30, 40])], [50], heads=(7, 1), seed=3)
    k, v = odd(x.k), odd(x.v)
    plan = PrefixPlan(x.q, k[1], v[1], x.bt, x.ctx, x.groups, x.scale, x.max_ctx)
    want = plan(x.q, x.k, x.v)
    check(want, x)
    assert torch.equal(plan(x.q, k[1], v[1]), want) and torch.equal(plan.run_layer(1, x.q, k, v), want)
    plan = DecodePlan(x.q, x.k, x.v, x.bt, x.ctx, x.scale, x.max_ctx)
    want = plan()
    assert torch.equal(plan.run_layer(1, x.q, k, v), want)
    c = Case([(70, 6), (300, 2)], (7, 1, 64), seed=4)
    k, v = odd(c.k), odd(c.v)
    plan = TreePlan(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes)
    want = plan(c.q, c.k, c.v)
    assert torch.equal(plan(c.q, k[1], v[1]), want) and torch.equal(plan.run_layer(1, c.q, k, v), want)
    for bad in (k[:, :, ::2], k.expand(2, 1, -1, -1, -1)[..., :32]):
        with pytest.raises(ValueError):
            plan.run_layer(1, c.q, bad, bad)
