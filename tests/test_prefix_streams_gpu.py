"""A shared-prefix plan that is dropped while its calls on another stream are still to run: its work list stays theirs."""

import pytest
import torch

from engine.hip_prefix import PrefixPlan
from prefix_cases import batch, check

pytestmark = pytest.mark.gpu


def test_a_plan_dropped_before_its_calls_have_run():
    x = batch([(512, [100] * 4), (64, [9, 20])], [300], seed=21)
    x.max_ctx = 612

    def plan():
        return PrefixPlan(x.q, x.k, x.v, x.bt, x.ctx, x.groups, x.scale, x.max_ctx, host_context_lens=x.lens)

    want = plan()(x.q, x.k, x.v)
    check(want, x)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        p = plan()
        n, at = p._list.numel(), p._list.data_ptr()
        with torch.cuda.stream(s):
            torch.cuda._sleep(20_000_000)  # the call is still to run when the plan is gone
            out = p(x.q, x.k, x.v)
        del p
        later = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(8)]
        assert at not in [t.data_ptr() for t in later]
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del later
    # on its own stream memory is handed on in order, without waiting
    p = plan()
    out = p(x.q, x.k, x.v)
    del p
    later = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and len(later) == 8
