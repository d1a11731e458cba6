"""Tree attention over values far from 1: small and large V through split runs, infinities beside large values, scores that
rise along the keys, and sums that cancel. The bounds are the kernel's own roundings, tighter than tree_cases'."""

import numpy as np
import pytest
import torch

from engine.hip_tree import paged_tree_attention
from tree_cases import Case

HEADS = {"64": (14, 2, 64), "64rows": (4, 2, 64), "128": (12, 2, 128)}


def attend(c: Case, **kw):
    return paged_tree_attention(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes,
                                quant=c.quant(), **kw)


def rows(c: Case):
    """(row, head, visible keys' K, V in float64, q) of every row that sees a key."""
    q, k, v = c.q.cpu().double(), c.k.cpu().double(), c.v.cpu().double()
    if c.ks is not None:
        k, v = k * c.ks.cpu().double()[..., None], v * c.vs.cpu().double()[..., None]
    at = 0
    for i, (start, n) in enumerate(c.seqs):
        ids = c.bt[i, :-(-(start + n) // c.B)].cpu().long()
        kk, vv = (t[:, ids].reshape(c.Hkv, -1, c.D) for t in (k, v))
        for r in range(n):
            on = torch.tensor(list(range(start)) + sorted(start + a for a in c.sets[at + r] if a < n), dtype=torch.long)
            for h in range(c.Hq if len(on) else 0):
                g = h // (c.Hq // c.Hkv)
                yield at + r, h, kk[g, on], vv[g, on], q[at + r, h]
        at += n


def reference(c: Case):
    """(out, tol) in 64 bits. With eps of the sum of p |v|:
    - p enters as two bf16 terms: the first cut off leaves less than 2^-7 p, the second rounds that by 2^-8: 2^-15, and as
      much in the denominator (plain pools sum these values); the second is taken of p (1 + 2^-20);
    - the score is an fp32 sum of D products, scaled, with a maximum taken away, and a split's maximum another: (D + 16)
      roundings of 2^-24 of the largest sum |q k| scale; the exponential 2^-22; both twice, for the denominator;
    - n keys are summed 32 (a matrix instruction's) at a time: n / 16 + 64 additions of two terms, 2^-24 each, twice;
    - splits are joined in fp32: 128 of them and a few products, 2^-24 each;
    and the result is rounded to bf16, 2^-8 of it."""
    out = torch.zeros(c.q.shape, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for t, h, k, v, q in rows(c):
        p = torch.softmax(k @ q * c.scale, 0)
        size = (k.abs() @ q.abs()).max() * c.scale
        out[t, h] = p @ v
        eps = 2.0 ** -14 + 2.0 ** -20 + 2 * ((c.D + 16) * 2.0 ** -24 * size + 2.0 ** -22) + \
            2 * (len(p) / 16 + 64) * 2.0 ** -24 + 136 * 2.0 ** -24
        tol[t, h] = eps * (p @ v.abs()) + 2.0 ** -8 * out[t, h].abs()
    return out, tol


def check(got, ref, scale=1.0):
    out, tol = ref
    worst = ((got.cpu().double() - out * scale).abs() - tol * scale).max().item()  # NaN for NaN
    assert worst <= 0, f"past the bound by {worst / scale} x {scale}"


def positions(c: Case, i: int):
    """(blocks, offsets) of sequence i's keys."""
    p = torch.arange(sum(c.seqs[i]), device=c.bt.device)
    return c.bt[i].long()[p // c.B], p % c.B


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_small_and_large_values_in_splits(heads, int8):
    """V times a power of two gives the result times it, whatever the number of splits."""
    c = Case([(700, 5), (90, 9), (1300, 1)], HEADS[heads], int8=int8, seed=31, scale_dtype=torch.float32)
    ref = reference(c)
    v, vs = c.v, c.vs
    for e in (-100, -30, -24, -20, -16, -14, 0, 15, 16, 30, 100):
        c.v, c.vs = (v, vs * 2.0 ** e) if int8 else (v * 2.0 ** e, None)
        for splits in (1, 2, 5, None):
            check(attend(c, num_splits=splits), ref, 2.0 ** e)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
def test_rows_of_small_and_large_channels(heads):
    """Channels 2^-60 to 2^60 side by side, each within its own bound."""
    c = Case([(700, 5), (90, 9)], HEADS[heads], seed=32)
    c.v *= torch.exp2(torch.linspace(-60, 60, c.D, device="cuda").round()).bfloat16()
    ref = reference(c)
    for splits in (1, 4):
        check(attend(c, num_splits=splits), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("splits", [1, 2, 6])
def test_an_infinite_channel_beside_large_finite_ones(heads, splits):
    c = Case([(900, 4)], HEADS[heads], seed=33)
    c.v *= 3e5
    ref = reference(c)
    blocks, offsets = positions(c, 0)
    c.v[:, blocks[200], offsets[200], 5] = float("inf")
    got = attend(c, num_splits=splits)
    assert (got[..., 5] == float("inf")).all()
    keep = [i for i in range(c.D) if i != 5]
    check(got[..., keep], (ref[0][..., keep], ref[1][..., keep]))


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("step", [3.0, 7.0, 13.0, -13.0, 40.0])
def test_scores_that_rise_along_the_keys(heads, int8, step):
    """Scores that grow by `step` (natural logarithm) every 64 keys: the running maximum is raised in later stages too, by
    less and by more than the kernel lets it lag (2^16), and the sums so far shrink by factors between 0 and 1."""
    c = Case([(1000, 6), (333, 20)], HEADS[heads], int8=int8, seed=34)
    # channel 0: 8 in every q, and level times 1 / (8 scale) in K
    c.q[..., 0] = 8
    for i in range(2):
        blocks, offsets = positions(c, i)
        level = (torch.arange(len(blocks), device="cuda") / 64) * step / (8 * c.scale)
        if not int8:
            c.k[:, blocks, offsets, 0] = level.bfloat16()
        else:  # the row's largest, in a scale of its own: the other channels keep their values within a step
            x = c.k[:, blocks, offsets].float() * c.ks[:, blocks, offsets].float()[..., None]
            x[..., 0] = level
            s = (x.abs().amax(-1) / 127).half()
            c.k[:, blocks, offsets] = (x / s.float()[..., None]).round().clamp(-127, 127).to(torch.int8)
            c.ks[:, blocks, offsets] = s
    ref = reference(c)
    for splits in (1, 3):
        check(attend(c, num_splits=splits), ref)


def cancelling(c: Case):
    """Keys in pairs of almost the same K and opposite V: the results are a few percent of the sums of p |v|."""
    g = torch.Generator().manual_seed(5)
    for i in range(len(c.seqs)):
        blocks, offsets = positions(c, i)
        n = len(blocks) // 2 * 2
        a, b = (blocks[0:n:2], offsets[0:n:2]), (blocks[1:n:2], offsets[1:n:2])
        k = c.k[:, a[0], a[1]]
        if c.ks is None:
            c.k[:, b[0], b[1]] = k * (1 + 2.0 ** -6 * torch.randint(0, 3, k.shape, generator=g).to(k.device)).to(k.dtype)
        else:
            c.k[:, b[0], b[1]] = (k + torch.randint(-1, 2, k.shape, generator=g).to(k)).clamp(-127, 127)
            for s in (c.ks, c.vs):
                s[:, b[0], b[1]] = s[:, a[0], a[1]]
        c.v[:, b[0], b[1]] = -c.v[:, a[0], a[1]]


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_cancelling_sums(heads, int8):
    c = Case([(400, 5), (31, 9), (1200, 2)], HEADS[heads], int8=int8, seed=35)
    cancelling(c)
    ref = reference(c)
    for splits in (1, 4):
        check(attend(c, num_splits=splits), ref)


def bf16(x):
    return x.float().bfloat16().double()


@pytest.mark.parametrize("terms,within", [(2, True), (1, False)])
def test_the_bound_tells_one_bf16_term_from_two(terms, within):
    """The bound on the CPU: probabilities cut to two bf16 terms keep it, rounded to one they do not."""
    c = Case([(400, 5), (31, 9)], HEADS["64"], seed=35, device="cpu")
    cancelling(c)
    out, tol = reference(c)
    worst = -np.inf
    for t, h, k, v, q in rows(c):
        z = k @ q * c.scale
        p = torch.exp(z - z.max())
        if terms == 2:
            cut = (p.float().view(torch.int32) & -65536).view(torch.float32).double()
            p = cut + bf16(p * (1 + 2.0 ** -20) - cut)
        else:
            p = bf16(p)
        worst = max(worst, ((bf16(p @ v / p.sum()) - out[t, h]).abs() - tol[t, h]).max().item())
    assert (worst <= 0) == within, worst
