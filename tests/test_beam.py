"""The selection over beams and vocabulary against 64 bits, on the CPU and the GPU: ties, masked and broken rows, logits in any
order, ragged requests."""

import math

import numpy as np
import pytest
import torch

from engine.hip_beam import beam_select, copy_blocks

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def expected(logits, scores, bounds, n):
    """float64 scores, beams and tokens [groups, n], from the definition: a row's tokens in the order of their logits, rows
    against each other by the scores."""
    l, cum = logits.double().cpu().numpy(), scores.double().cpu().numpy()
    G = len(bounds) - 1
    score, beam, token = np.full((G, n), -np.inf), np.full((G, n), -1), np.full((G, n), -1)
    for g in range(G):
        found = []
        for b in range(max(0, min(bounds[g + 1], len(l)) - bounds[g])):
            row = l[bounds[g] + b]
            if np.isnan(row).any() or not row.max() < np.inf or row.max() == -np.inf or not np.isfinite(cum[bounds[g] + b]):
                continue
            off = cum[bounds[g] + b] - (row.max() + np.log(np.exp(row - row.max()).sum()))
            order = np.argsort(-row, kind="stable")[:n]
            found += [(-(off + row[t]), b, rank, int(t)) for rank, t in enumerate(order) if row[t] > -np.inf]
        for i, (z, b, _, t) in enumerate(sorted(found)[:n]):
            score[g, i], beam[g, i], token[g, i] = -z, b, t
    return score, beam, token


def check(logits, scores, beams, n, bounds=None):
    got = beam_select(logits, scores, beams, n)
    if bounds is None:
        bounds = list(range(0, logits.shape[0] + 1, beams))
    score, beam, token = expected(logits, scores, bounds, n)
    assert np.array_equal(got.beams.cpu().numpy(), beam)
    assert np.array_equal(got.tokens.cpu().numpy(), token)
    s = got.scores.double().cpu().numpy()
    # rounded once (2^-24); the exponentials are off by 2^-22 each, and eight of them added up by 7 2^-24: 2^-20 of their sum
    none = np.isneginf(score)
    assert np.array_equal(none, np.isneginf(s))
    s, score = s[~none], score[~none]
    assert (np.abs(s - score) <= np.abs(score) * 2 ** -24 + 2 ** -20).all()


def rand(R, V, dtype, device, seed=0, spread=3.):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * spread).to(dtype).to(device), (-9 * torch.rand(R, generator=g)).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,V,beams,n", [(1, 1, 1, 1), (2, 7, 2, 3), (4, 7, 2, 64), (6, 1001, 3, 6), (4, 151936, 4, 8),
                                         (12, 32003, 1, 10), (30, 4099, 5, 33), (8, 2048, 8, 64), (64, 513, 64, 1),
                                         (600, 777, 4, 5), (520, 20011, 4, 16)])
def test_sizes(device, dtype, R, V, beams, n):
    if device == "cpu" and R * V > 10 ** 6:
        R = beams
    logits, scores = rand(R, V, dtype, device, seed=R + V)
    check(logits, scores, beams, n)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 8, 64])
def test_ties_go_to_the_lowest_row_then_token(device, dtype, n):
    """Logits of few values, rows that are equal, all logits equal."""
    g = torch.Generator().manual_seed(n)
    logits = torch.randint(0, 4, (6, 5003), generator=g).to(dtype).to(device)
    logits[3] = logits[2]
    scores = torch.tensor([0., -1., -2., -2., -2.5, -2.5]).to(device)
    check(logits, scores, 3, n)
    check(logits, torch.zeros(6, device=device), 6, n)
    check(torch.full((6, 30011), 2.5, dtype=dtype, device=device), torch.zeros(6, device=device), 2, n)
    zeros = torch.zeros(2, 3000, dtype=dtype, device=device)
    zeros[:, ::3] = -0.
    check(zeros, torch.zeros(2, device=device), 2, n)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("down", [True, False])
def test_sorted_logits(device, down):
    """Vocabularies in the order of their frequency: the largest logits stand together, in one piece of a row or in one thread's
    part of it."""
    l = torch.linspace(-20, 20, 40000)
    logits = torch.stack([l, l / 2, l.roll(7), torch.repeat_interleave(l[::80], 80)])
    logits = (logits.flip(1) if down else logits).to(device)
    scores = torch.tensor([0., -0.25, -0.5, -1.]).to(device)
    for n in (1, 16, 64):
        check(logits, scores, 4, n)
        check(logits, scores, 2, n)


@pytest.mark.parametrize("device", DEVICES)
def test_masked_and_broken_rows(device):
    logits, scores = rand(12, 3001, torch.float32, device, seed=2)
    logits[0, 5:] = -math.inf           # five tokens left
    logits[1] = -math.inf               # none
    logits[2, :3000] = -math.inf        # the last one
    logits[3, 17] = math.nan
    logits[4, 18] = math.inf
    scores[5] = -math.inf               # a beam that has ended
    scores[6] = math.nan
    scores[7] = math.inf
    logits[8] *= 1e30
    logits[9] *= 1e-30
    for beams, n in ((1, 8), (2, 8), (3, 4), (12, 64)):
        check(logits, scores, beams, n)
    half = logits.clamp(-60000, 60000).half()
    half[1], half[3, 17], half[4, 18] = -math.inf, math.nan, math.inf
    check(half, scores, 6, 16)


@pytest.mark.parametrize("device", DEVICES)
def test_requests_of_different_numbers_of_beams(device):
    logits, scores = rand(19, 2003, torch.bfloat16, device, seed=4)
    for bounds in ([0, 4, 5, 5, 13, 19], [2, 3, 9], [0, 0], [0, 19], [7, 30], [0]):
        check(logits, scores, torch.tensor(bounds, dtype=torch.int32, device=device), 6, bounds)
    got = beam_select(logits, scores, torch.tensor([-5, 2, 1], dtype=torch.int32, device=device), 3)
    score, beam, token = expected(logits, scores, [0, 2], 3)  # clamped to the rows; a group that ends before it starts is empty
    assert np.array_equal(got.tokens[:1].cpu().numpy(), token) and (got.tokens[1] == -1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_rows_inside_wider_ones(device):
    wide, scores = rand(6, 1500, torch.float16, device, seed=5)
    for a, b in ((0, 1499), (1, 1500), (3, 1200)):
        check(wide[:, a:b], scores, 3, 7)
    check(wide[::2, 1:], scores[:3].contiguous(), 3, 7)
    check(wide[:1].expand(6, 1500), scores, 3, 7)  # the first step: every beam from one row


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows(device):
    got = beam_select(torch.empty(0, 9, device=device), torch.empty(0, device=device), 3, 4)
    assert got.scores.shape == got.beams.shape == got.tokens.shape == (0, 4)
    got = beam_select(torch.empty(0, 9, device=device), torch.empty(0, device=device),
                      torch.zeros(3, dtype=torch.int32, device=device), 4)
    assert (got.tokens == -1).all() and got.scores.isneginf().all() and got.tokens.shape == (2, 4)


@pytest.mark.parametrize("device", DEVICES)
def test_more_than_1024_beams_are_not_read(device):
    logits, scores = rand(1030, 5, torch.float32, device, seed=6)
    scores[1024:] = 100.
    got = beam_select(logits, scores, torch.tensor([0, 1030], dtype=torch.int32, device=device), 9)
    score, beam, token = expected(logits[:1024], scores[:1024], [0, 1024], 9)
    assert np.array_equal(got.beams.cpu().numpy(), beam) and np.array_equal(got.tokens.cpu().numpy(), token)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    logits, scores = rand(6, 100, torch.float32, device)
    starts = torch.tensor([0, 6], dtype=torch.int32, device=device)
    for l, s, b, n in ((logits[0], scores, 3, 4), (logits.double(), scores, 3, 4), (logits.T, scores, 3, 4), (logits[:, :0], scores, 3, 4),
                       (logits, scores[:5], 3, 4), (logits, scores.double(), 3, 4), (logits, scores, 0, 4), (logits, scores, 4, 4),
                       (logits, scores, 3, 0), (logits, scores, 3, 65), (logits, scores, starts.long(), 4),
                       (logits, scores, starts[None], 4), (logits, scores, starts[:0], 4), (logits, scores, 1025, 4)):
        with pytest.raises(ValueError):
            beam_select(l, s, b, n)
    if device == "cuda":
        with pytest.raises(ValueError):
            beam_select(logits, scores.cpu(), 3, 4)
        with pytest.raises(ValueError):
            beam_select(logits, scores, starts.cpu(), 4)


@pytest.mark.gpu
def test_captured_selections():
    logits, scores = rand(8, 30011, torch.bfloat16, "cuda", seed=7)
    beam_select(logits, scores, 4, 8)
    graphs = []
    for beams in (4, 8):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = beam_select(logits, scores, beams, 8)
        graphs.append((g, out, beams))
    for seed in range(4):
        other, more = rand(8, 30011, torch.bfloat16, "cuda", seed=20 + seed)
        logits.copy_(other)
        scores.copy_(more)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out, beams in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, beam_select(logits, scores, beams, 8)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,row", [(torch.bfloat16, (64,)), (torch.int8, (128,)), (torch.float16, ()), (torch.float32, (5,)),
                                       (torch.int8, (3,)), (torch.uint8, ())])
@pytest.mark.parametrize("L,H,B", [(1, 1, 16), (3, 2, 16), (28, 2, 32), (5, 7, 5)])
def test_copies_on_the_gpu(dtype, row, L, H, B):
    g = torch.Generator().manual_seed(L * 7 + B)
    n, N = 300, 640
    shape = (L, H, N, B, *row)
    make = lambda: (torch.randint(0, 100, shape, generator=g).to(dtype)).cuda()  # noqa: E731
    ids = torch.randperm(N, generator=g)[:2 * n].view(2, n).tolist()
    copies = [(s, d, int(torch.randint(0, B + 1, (), generator=g))) for s, d in zip(*ids)]
    copies.append((copies[0][0], next(i for i in range(N) if i not in ids[0] + ids[1]), B))  # one source twice
    for count in (1, 2, 301):
        pools = [make(), make()]
        want = [t.clone() for t in pools]
        for t in want:
            for s, d, k in copies[:count]:
                t[:, :, d, :k] = t[:, :, s, :k]
        copy_blocks(pools, copies[:count])
        assert all(torch.equal(a, b) for a, b in zip(pools, want))


@pytest.mark.gpu
def test_copies_in_layers_that_lie_apart():
    both = torch.randn(4, 2, 3, 9, 16, 64, device="cuda").bfloat16()  # K and V side by side
    want = both.clone()
    want[:, :, :, 5, :7] = want[:, :, :, 2, :7]
    copy_blocks((both[:, 0], both[:, 1]), [(2, 5, 7)])
    assert torch.equal(both, want)
    with pytest.raises(ValueError):
        copy_blocks((both[:, 0], both[:, 1]), [(2, 5, 7), (3, 5, 7)])
    assert torch.equal(both, want)


@pytest.mark.gpu
def test_captured_copies():
    pool = torch.randn(4, 2, 9, 16, 64, device="cuda")
    copy_blocks((pool,), [(0, 1, 16)])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        copy_blocks((pool,), [(2, 5, 7), (2, 6, 3)])
    for _ in range(3):
        pool.normal_()
        want = pool.clone()
        want[:, :, 5, :7], want[:, :, 6, :3] = want[:, :, 2, :7], want[:, :, 2, :3]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, want)
