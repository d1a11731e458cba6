"""Rows of the logits that belong to no sequence: before the first one's, behind the last one's, and with query starts past the
rows. They come out as they went in."""

import pytest
import torch

from engine.hip_logits import LogitsRules

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("starts", [[0, 2, 3], [3, 5, 9], [2, 2, 4], [5, 12, 12], [12, 12, 12], [0, 0, 0], [11, 12, 40], [4, 30, 50],
                                    [20, 30, 40]])
@pytest.mark.parametrize("vocab", [17, 5003])
def test_rows_of_no_sequence_are_copied(device, dtype, starts, vocab):
    rules = LogitsRules(vocab, 2, bias_tokens=torch.tensor([3, 4], dtype=torch.int32, device=device),
                        bias_values=torch.tensor([8.0, 16.0], device=device),
                        bias_starts=torch.tensor([0, 1, 2], dtype=torch.int32, device=device))
    l = torch.randint(-8, 8, (12, vocab), generator=torch.Generator().manual_seed(1)).to(dtype).to(device)
    q = torch.tensor(starts, dtype=torch.int32, device=device)
    want = l.clone()
    for s, (token, value) in enumerate(((3, 8), (4, 16))):
        want[min(starts[s], 12):min(starts[s + 1], 12), token] += value
    out = torch.full_like(l, float("nan"))
    assert torch.equal(rules.apply(l, query_starts=q, out=out), want)
    assert torch.equal(rules.apply(l, query_starts=q), want)
    assert torch.equal(rules.apply(l, query_starts=q, out=l), want)
