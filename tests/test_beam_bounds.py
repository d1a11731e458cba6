"""How far a row's log-sum may be from 64 bits: rows whose weight lies where the exponentials' arguments are rounded most."""

import numpy as np
import pytest
import torch

from engine.hip_beam import beam_select

# Of the terms exp(-d) below a piece's largest logit: the argument is off by d 2^-22.8 (difference, constant, product), exp2 by
# 2^-23, sums of eight by 7 2^-24; the weighted mean of d is W(16384 / e) = 6.8 at most: 2^-19.4 together.
BOUND = 2.0 ** -19
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def rows(dtype, V, top, R=96):
    """One logit at `top`, the others some depth below it, one depth a row, around log(V) - log(log(V))."""
    g = torch.Generator().manual_seed(V)
    depth = 4 + 8 * torch.rand(R, 1, generator=g, dtype=torch.float64)
    l = (top - depth).expand(R, V).clone()
    l[torch.arange(R), torch.randint(0, V, (R,), generator=g)] = top
    return l.to(dtype)


def log_sums(l):
    l = l.double().numpy()
    m = l.max(-1, keepdims=True)
    return m[:, 0] + np.log(np.exp(l - m).sum(-1))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1000, 16384, 151936])
@pytest.mark.parametrize("top", [0.0, 11.3])
def test_log_sums(device, dtype, V, top):
    l = rows(dtype, V, top, 96 if device == "cuda" else 8)
    got = beam_select(l.to(device), torch.zeros(l.shape[0], device=device), 1, 1)
    best, at = l.max(-1)
    assert torch.equal(got.tokens[:, 0].cpu(), at)
    want = best.double().numpy() - log_sums(l)
    assert (np.abs(got.scores[:, 0].double().cpu().numpy() - want) <= np.abs(want) * 2 ** -24 + BOUND).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_order_of_rows(device, dtype):
    """Rows whose best candidates are twice the bound apart, and the scores' own rounding to fp32: in the order of 64 bits."""
    V, R = 40000, 64
    l = rows(dtype, V, 3.0, R)
    sums = log_sums(l)
    best = l.max(-1).values.double().numpy()
    # best candidates that ascend by 2^-17 with the row: more than 2 BOUND, and 2^-23 for the scores given
    cum = torch.from_numpy(sums - best - 1 + np.arange(R) * 2.0 ** -17).float()
    got = beam_select(l.to(device), cum.to(device), R, 1)
    want = cum.double().numpy() + best - sums
    assert np.sort(want)[-1] - np.sort(want)[-2] > 2 * BOUND and int(got.beams[0, 0]) == int(want.argmax()) == R - 1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_equal_rows_tie(device, dtype):
    l = rows(dtype, 20011, 2.0, 4).repeat_interleave(3, 0)
    for n in (1, 9, 40):
        got = beam_select(l.to(device), torch.full((12,), -2.5, device=device), 3, n)
        for g in range(4):
            k = n // 3 * 3
            s = got.scores[g].cpu()
            assert got.beams[g].cpu()[:3].tolist() == [0, 1, 2][:n] and (s[:k:3] == s[2:k:3]).all()
