"""Where LogitsRules.apply may write: over the logits themselves or beside them, never over other rows of theirs, which the
kernel's workgroups may still have to read."""

import pytest
import torch

from engine.hip_logits import LogitsRules

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
V, R = 1003, 4


def rules(device):
    return LogitsRules(V, R, presence=torch.full((R,), 0.5, device=device),
                       history=torch.arange(R, dtype=torch.int32, device=device),
                       history_starts=torch.arange(R + 1, device=device))


@pytest.mark.parametrize("device", DEVICES)
def test_overlapping_outputs_are_refused(device):
    r = rules(device)
    wide = torch.randn(R + 2, 3 * V, device=device)
    flat = wide.view(-1)
    view = lambda at, stride: torch.as_strided(flat, (R, V), (stride, 1), at)  # noqa: E731
    logits = view(0, V)
    for out in (view(V, V), view(1, V), view(V - 1, V), view(3 * V, V), view(0, 2 * V), view(0, 0), view(8 * V, V - 1),
                torch.zeros(1, V, device=device).expand(R, V)):
        before = flat.clone()
        with pytest.raises(ValueError, match="overlap"):
            r.apply(logits, out=out)
        assert torch.equal(flat, before)
    with pytest.raises(ValueError, match="overlap"):
        r.apply(view(0, 0), out=view(0, 0))


@pytest.mark.parametrize("device", DEVICES)
def test_outputs_beside_the_logits(device):
    r = rules(device)
    wide = torch.randn(2 * R + 2, 3 * V, device=device)
    flat, fresh = wide.view(-1), wide.clone()
    view = lambda at, stride: torch.as_strided(flat, (R, V), (stride, 1), at)  # noqa: E731
    for a, b in ((view(0, V), view(R * V, V)), (view(R * V, V), view(0, V)), (view(0, 3 * V), view(V, 3 * V)),
                 (view(V, 2 * V), view(0, 2 * V)), (view(0, 0), view(V, V)), (view(0, V), view(R * V, 2 * V)),
                 (view(5, V), view(5, V))):
        wide.copy_(fresh)
        want = r.apply(a.contiguous().clone())
        assert r.apply(a, out=b).data_ptr() == b.data_ptr()
        assert torch.equal(b, want)
    one = LogitsRules(V, 1, presence=torch.ones(1, device=device))
    assert torch.equal(one.apply(flat[:V].view(1, V), out=flat[V:2 * V].view(1, V)), flat[:V].view(1, V))
