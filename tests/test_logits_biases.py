"""Bias lists as ban and allow lists make them: runs of neighbouring tokens, the whole vocabulary, tokens named many times,
each summed in the list's order."""

import numpy as np
import pytest
import torch

from engine.hip_logits import LogitsRules

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def lists(kind, V, rng):
    """Two sequences' lists of tokens."""
    if kind == "run":  # more neighbours than a workgroup's tile holds
        return [np.arange(3000, 7096), np.arange(V - 300, V)]
    if kind == "all":
        return [rng.permutation(V), np.arange(V)[::-1]]
    if kind == "twice":  # every token of a range two to five times, in any order
        return [np.concatenate([rng.permutation(1500) + 100 for _ in range(5)]), np.repeat(np.arange(40, 700), 2)]
    if kind == "one":
        return [np.full(2500, 4321), np.concatenate([np.full(300, 5), np.arange(900), np.full(300, 5)])]
    return [rng.randint(-3, V + 3, 5000), np.zeros(0, dtype=int)]  # some outside the vocabulary


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["run", "all", "twice", "one", "outside"])
def test_long_lists(device, dtype, kind):
    """Equal to the sums in fp32, one entry after the other, and one more sum with the logit: one result, no bound."""
    V, rng = 9001, np.random.RandomState(len(kind))
    ts = lists(kind, V, rng)
    xs = [(rng.randn(len(t)) * 10.0 ** rng.randint(-4, 5, len(t))).astype(np.float32) for t in ts]
    l = torch.randn(5, V, generator=torch.Generator().manual_seed(1)).to(dtype)
    rules = LogitsRules(V, 2, bias_tokens=torch.from_numpy(np.concatenate(ts)).int().to(device),
                        bias_values=torch.from_numpy(np.concatenate(xs)).to(device),
                        bias_starts=torch.tensor([0, len(ts[0]), len(ts[0]) + len(ts[1])], dtype=torch.int32, device=device))
    got = rules.apply(l.to(device), query_starts=torch.tensor([0, 2, 5], dtype=torch.int32, device=device)).cpu()
    for s, rows in ((0, slice(0, 2)), (1, slice(2, 5))):
        sums = np.zeros(V, dtype=np.float32)
        inside = (ts[s] >= 0) & (ts[s] < V)
        np.add.at(sums, ts[s][inside], xs[s][inside])  # in the order given
        assert torch.equal(got[rows], (l[rows].float() + torch.from_numpy(sums)).to(dtype)), s


@pytest.mark.parametrize("device", DEVICES)
def test_long_lists_beside_the_other_rules(device):
    V, rng = 5000, np.random.RandomState(3)
    tokens, values = rng.permutation(V)[:4096], rng.randn(4096).astype(np.float32)
    history, l = rng.randint(0, V, 3000), torch.randn(3, V, generator=torch.Generator().manual_seed(2))
    i32 = lambda x: torch.from_numpy(np.asarray(x)).int().to(device)  # noqa: E731
    path = torch.tensor([1, 2, 2], device=device)
    rules = LogitsRules(V, 1, history=i32(history), history_starts=torch.tensor([0, 3000], device=device),
                        frequency=torch.tensor([0.5], device=device), bias_tokens=i32(tokens),
                        bias_values=torch.from_numpy(values).to(device), bias_starts=i32([0, 4096]))
    got = rules.apply(l.to(device), query_starts=i32([0, 3]), tokens=path,
                      masks=torch.tensor([[1], [3], [7]], device=device)).cpu().double()
    for r, seen in enumerate(([1], [1, 2], [1, 2, 2])):
        count = np.bincount(np.concatenate([history, seen]), minlength=V)
        bias = np.zeros(V)
        bias[tokens] = values
        want = l[r].double() - torch.from_numpy(0.5 * count) + torch.from_numpy(bias)
        # two sums in fp32 of values below 8
        assert ((got[r] - want).abs() <= 2 * 2.0 ** -24 * 8).all()
