"""Tree maps of a step with room for more nodes than it has (sipa_tree_maps with fill_rest): the rows behind the last
sequence's nodes get a slot, a position and no ancestors of their own, so that a captured step may store every row."""

import ctypes

import numpy as np
import pytest
import torch

from engine import _hip
from engine.hip_quant import store_layer
from engine.hip_tree import tree_maps
from test_tree_capi import maps as params

gpu = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Step:
    """S sequences on blocks of 16 and a scratch block, with room for T nodes."""

    def __init__(self, S=4, T=40, seed=0):
        self.S, self.T, self.blocks = S, T, S * 4 + 1
        rng = np.random.RandomState(seed)
        self.rest_slot = (self.blocks - 1) * 16 + 5
        self.table = i32(rng.permutation(self.blocks - 1).reshape(S, 4))
        self.rows, self.starts, self.counts = i32(range(S)), i32([0] * S), i32([0] * S)
        self.parents = i32([-1] * T)

    def set(self, starts, trees):
        flat = [p for t in trees for p in t]
        self.starts.copy_(i32(starts)), self.counts.copy_(i32([len(t) for t in trees]))
        self.parents.copy_(i32(flat + [-1] * (self.T - len(flat))))
        return len(flat)

    def run(self, rest=True, **kw):
        return tree_maps(self.table, self.rows, self.starts, self.counts, self.parents, 16, 4, 16,
                         rest_slot=self.rest_slot if rest else None, **kw)

    def check(self, m, live):
        exact = tree_maps(self.table, self.rows, self.starts, self.counts, self.parents[:live], 16, 4, 16) if live else None
        for name, want in (("positions", 0), ("slots", self.rest_slot), ("slot_blocks", self.rest_slot // 16),
                           ("slot_offsets", self.rest_slot % 16), ("masks", 0)):
            got = getattr(m, name)
            assert (got[live:] == want).all(), name
            assert exact is None or torch.equal(got[:live], getattr(exact, name)), name
        for name in ("query_starts", "context_lens", "last_rows", "block_tables"):
            assert exact is None or torch.equal(getattr(m, name), getattr(exact, name)), name


STEPS = [([3, 20, 0, 41], [[-1, 0, 1, 0], [-1], [-1, 0, -1], [-1, 0, 1, 2, 3, 4]]),
         ([7, 21, 3, 47], [[-1], [], [-1, -1], []]),
         ([8, 22, 5, 48], [list(range(-1, 9))] * 4),  # all 40 rows
         ([0, 0, 0, 0], [[], [], [], []]),
         ([18, 32, 15, 58], [[-1, 0], [-1, 0, 0], [], [-1]])]


@gpu
@pytest.mark.parametrize("T", [40, 300])
def test_rows_behind_have_values(T):
    s = Step(T=T)
    for starts, trees in STEPS:
        live = s.set(starts, trees)
        s.check(s.run(), live)


@gpu
def test_without_a_slot_the_rows_behind_stay():
    s = Step()
    out = s.run()
    live = s.set(*STEPS[0])
    for t in out:
        t.fill_(-5)
    s.run(rest=False, out=out)
    for t in (*out[:4], out.masks):
        assert (t[live:] == -5).all() and (t[:live] != -5).any()


@gpu
def test_a_captured_step_stores_every_row():
    """Replays of maps and a store over all rows, with fewer nodes than the replay before too: only the live nodes' slots and
    the scratch slot change."""
    s = Step()
    k, v = (torch.randn(s.T, 2, 64, device="cuda").bfloat16() for _ in range(2))
    pools = [torch.zeros(1, 2, s.blocks, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    out = s.run()
    store_layer(0, k, v, out.slot_blocks, out.slot_offsets, *pools)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.run(out=out)
        store_layer(0, k, v, out.slot_blocks, out.slot_offsets, *pools)
    for starts, trees in STEPS:
        live = s.set(starts, trees)
        k.normal_(), v.normal_()
        before = [p.clone() for p in pools]
        g.replay()
        torch.cuda.synchronize()
        s.check(out, live)
        for p, b, x in zip(pools, before, (k, v)):
            flat, want = p[0].reshape(2, -1, 64), b[0].reshape(2, -1, 64)
            want[:, out.slots[:live]] = x[:live].transpose(0, 1)
            keep = torch.arange(s.blocks * 16, device="cuda") != s.rest_slot
            assert torch.equal(flat[:, keep], want[:, keep])


@gpu
def test_a_negative_slot_is_refused():
    s = Step()
    s.set(*STEPS[0])
    s.rest_slot = -1
    with pytest.raises(ValueError):
        s.run()


def test_the_library_refuses_a_negative_slot():
    assert _hip.lib().sipa_tree_maps(ctypes.byref(params(fill_rest=1, rest_slot=-1)), None) == _hip.EINVAL
