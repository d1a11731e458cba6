"""Copies of blocks in caches with per-channel K scales: a list that is refused leaves the staging slots as they were. CPU."""

import pytest
import torch

from engine import quant_cache
from engine.block_manager import BlockManager
from engine.config import ModelConfig
from engine.paged_cache import build_metadata
from engine.quant_cache import QuantPagedKVCache

CFG = ModelConfig(vocab_size=37, hidden_size=28, intermediate_size=24, num_layers=2, num_q_heads=7, num_kv_heads=1, head_dim=4)


def filled(tokens=6, n_stage=4):
    """A cache of blocks of four tokens and its manager, with one sequence written."""
    m = BlockManager(20, 4)
    cache = QuantPagedKVCache(CFG, 20, 4, "cpu", torch.float32, "gather", fmt="int8-kchannel", manager=m, n_stage=n_stage)
    m.allocate(0, tokens)
    write(cache, m, 0, 0, tokens)
    return m, cache


def write(cache, m, seq, start, n):
    cache.begin(n, build_metadata(m, [(seq, start, n)], "cpu"))
    for layer in range(2):
        cache.write(layer, *(torch.randn(n, 1, 4) for _ in range(2)))


def slots(cache):
    return dict(cache._stage_of), list(cache._free_stage)


@pytest.mark.parametrize("copies", [[(1, 5, 2), (1, 5, 2)], [(1, 5, 2), (5, 6, 2)], [(1, 20, 2)], [(1, 5, 2), (-1, 6, 1)], [(1, 5, 5)],
                                    [(1, 5, -1)], [(1, 1, 2)], [(1, 5)], [(1, 5, 1 << 40)]])
def test_refused_copies_change_nothing(copies):
    m, cache = filled()
    before, pools = slots(cache), [t.clone() for t in (cache.v, cache.v_scale, cache.stage)]
    with pytest.raises(ValueError):
        cache.copy_blocks(copies)
    assert slots(cache) == before
    assert all(torch.equal(a, b) for a, b in zip(pools, (cache.v, cache.v_scale, cache.stage)))


def test_copies_that_fail_give_their_slots_back(monkeypatch):
    m, cache = filled()
    before = slots(cache)

    def fail(pools, copies):
        raise RuntimeError("no launch")

    monkeypatch.setattr(quant_cache, "copy_blocks", fail)
    with pytest.raises(RuntimeError, match="no launch"):
        cache.copy_blocks([(1, 5, 2), (1, 6, 2)])
    assert slots(cache) == before


def test_copies_that_are_taken():
    m, cache = filled()
    copies = m.fork(0, [1, 2])
    cache.copy_blocks(copies)
    assert set(cache._stage_of) == {1} | {d for _, d, _ in copies} and len(cache._free_stage) == 1
    for _, d, n in copies:
        assert torch.equal(cache.stage[:, :, cache._stage_of[d], :n], cache.stage[:, :, cache._stage_of[1], :n])
        assert torch.equal(cache.v[:, :, d, :n], cache.v[:, :, 1, :n])
    cache.copy_blocks([])
    for s in (0, 1, 2):
        m.free(s)
    assert not cache._stage_of and len(cache._free_stage) == 4


def state(m):
    return {s: (m.block_table(s), m.seq_len(s)) for s in m.seq_ids()}, m.num_free_blocks(), m.num_shared_blocks()


def test_forks_without_staging_slots_are_refused_before_they_are_made():
    m, cache = filled(n_stage=3)
    before = state(m), slots(cache)
    with pytest.raises(RuntimeError, match="staging slots"):
        m.fork(0, [1, 2, 3])
    assert (state(m), slots(cache)) == before
    m.check_invariants()
    cache.copy_blocks(m.fork(0, [1, 2]))  # as many as there are
    assert not cache._free_stage
    m.allocate(7, 4)  # whole blocks are not staged
    write(cache, m, 7, 0, 4)
    assert m.fork(7, [8]) == []
    m.append_slots(8, 1)  # a last block that has not been written holds no slot
    cache.copy_blocks(m.fork(8, [9]))
    m.check_invariants()


def test_reorders_without_staging_slots_are_refused_before_they_are_made():
    m, cache = filled(n_stage=2)
    m.allocate(1, 4)
    write(cache, m, 1, 0, 4)
    cache.copy_blocks(m.fork(0, [2]))  # both slots are taken
    before = state(m), slots(cache)
    with pytest.raises(RuntimeError, match="staging slots"):
        m.reorder([0, 1], [0, 0])
    with pytest.raises(RuntimeError, match="staging slots"):
        m.reorder([0, 1, 2], [0, 0, 0])  # two copies, of which one slot comes back
    assert (state(m), slots(cache)) == before
    m.check_invariants()
    copies = m.reorder([0, 2], [0, 0])  # sequence 2's slot goes to its copy
    assert len(copies) == 1
    cache.copy_blocks(copies)
    assert m.reorder([0, 1], [1, 1]) == []  # nothing to copy
    copies = m.reorder([1, 2], [1, 1])  # sequence 1 goes on from 2: the slot that sequence 0 gave up serves the copy
    cache.copy_blocks(copies)
    assert set(cache._stage_of) == {b for c in copies for b in c[:2]} and not cache._free_stage
    for s in (0, 1, 2):
        m.free(s)
    assert not cache._stage_of and len(cache._free_stage) == 2
    m.check_invariants()


def test_forks_count_the_slots_of_copies_that_are_still_to_be_made():
    """Copies of several forks made in one call: the second fork finds the slots that the first one's copies will take."""
    m, cache = filled(n_stage=3)
    m.allocate(7, 7)
    write(cache, m, 7, 0, 7)
    copies = m.fork(0, [1])
    before = state(m), slots(cache)
    with pytest.raises(RuntimeError, match="staging slots"):
        m.fork(7, [8])
    with pytest.raises(RuntimeError, match="staging slots"):
        m.fork(1, [8])
    assert (state(m), slots(cache)) == before
    copies += m.reorder([0, 7], [0, 0])  # the slot of sequence 7's block goes to its copy
    cache.copy_blocks(copies)
    assert set(cache._stage_of) == {1} | {d for _, d, _ in copies}
    for _, d, n in copies:
        assert torch.equal(cache.stage[:, :, cache._stage_of[d], :n], cache.stage[:, :, cache._stage_of[1], :n])
    m.free(1)  # a fork that is given up before its copies are made gives its slot back
    m.fork(0, [9])
    m.free(9)
    for s in (0, 7):
        m.free(s)
    assert not cache._stage_of and sorted(cache._free_stage) == [0, 1, 2]
    m.check_invariants()
