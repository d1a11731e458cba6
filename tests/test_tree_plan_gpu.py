"""TreePlan as an object that a program keeps: its own scales after other layers'."""

import pytest
import torch

from engine.hip_decode import QuantKV
from engine.hip_tree import TreePlan
from tree_cases import Case

pytestmark = pytest.mark.gpu
HEADS = (14, 2, 64)


def plan_of(c: Case, **kw):
    return TreePlan(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes, quant=c.quant(), **kw)


@pytest.mark.parametrize("splits", [1, 2])
def test_a_plans_own_scales_after_other_scales(splits):
    """Without scales a call uses the plan's, whatever calls before it were given: layers of pools, or other scales."""
    c = Case([(70, 6), (300, 2)], HEADS, int8=True, seed=41)
    plan = plan_of(c, num_splits=splits)
    want = plan(c.q, c.k, c.v)
    k, v = torch.stack([c.k, c.k]), torch.stack([c.v, c.v])
    scales = QuantKV(1, torch.stack([c.ks * 3, c.ks]), torch.stack([c.vs * 5, c.vs]))
    other = plan.run_layer(0, c.q, k, v, scales)
    assert not torch.equal(other, want)
    assert torch.equal(plan(c.q, c.k, c.v), want)
    assert torch.equal(plan(c.q, c.k, c.v, quant=QuantKV(1, c.ks * 3, c.vs * 5)), other)
    assert torch.equal(plan(c.q, c.k, c.v), want)
    assert torch.equal(plan.run_layer(1, c.q, k, v, scales), want)
    with pytest.raises(ValueError):
        plan.run_layer(0, c.q, k, v)  # the plan's scales are one layer's
    assert torch.equal(plan(c.q, c.k, c.v), want)
