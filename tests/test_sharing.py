"""Sequences that share blocks: forks and reordered beams in the block manager, what may be written and truncated, the copies
in the caches, and a beam search over them against sequences that share nothing. CPU."""

import random

import numpy as np
import pytest
import torch

from engine.block_manager import BlockManager, OutOfBlocks
from engine.config import ModelConfig
from engine.hip_beam import beam_select, copy_blocks
from engine.hip_prefix import shared_groups
from engine.model import Qwen2Model
from engine.paged_cache import PagedKVCache, build_metadata, build_tree_metadata
from engine.quant_cache import QuantPagedKVCache

CFG = ModelConfig(vocab_size=37, hidden_size=28, intermediate_size=24, num_layers=2, num_q_heads=7, num_kv_heads=1, head_dim=4)


def test_fork_shares_full_blocks_and_copies_the_last():
    m = BlockManager(20, 4)
    m.allocate(0, 10)
    assert m.fork(0, [5, 6]) == [(2, 3, 2), (2, 4, 2)]
    assert m.block_table(5) == [0, 1, 3] and m.block_table(6) == [0, 1, 4] and m.seq_len(6) == 10
    assert m.ref_count(0) == 3 and m.ref_count(2) == 1 and m.num_shared_blocks() == 2
    assert m.append_slots(5, 3) == [14, 15, 20] and m.block_table(0) == [0, 1, 2]
    m.check_invariants()
    m.free(0)
    m.free(6)
    assert m.num_shared_blocks() == 0 and m.ref_count(0) == 1
    m.check_invariants()


@pytest.mark.parametrize("n", [0, 8])
def test_fork_at_a_block_boundary_copies_nothing(n):
    m = BlockManager(3, 4)
    m.allocate(0, n)
    assert m.fork(0, [1, 2, 3]) == []
    assert m.num_free_blocks() == 3 - n // 4
    m.check_invariants()
    assert m.append_slots(1, 1) == [(n // 4) * 4]


def test_fork_and_reorder_refuse():
    m = BlockManager(4, 4)
    m.allocate(0, 6)
    m.fork(0, [1])
    before = (m.block_table(0), m.block_table(1), m.num_free_blocks())
    with pytest.raises(KeyError):
        m.fork(9, [2])
    for ids in ([1], [2, 2], [0]):
        with pytest.raises(ValueError):
            m.fork(0, ids)
    with pytest.raises(OutOfBlocks):
        m.fork(0, [2, 3])
    for ids, parents in (([0, 0], [0, 0]), ([0, 1], [0]), ([0, 1], [0, 2]), ([0, 1], [-1, 0])):
        with pytest.raises(ValueError):
            m.reorder(ids, parents)
    with pytest.raises(KeyError):
        m.reorder([0, 7], [0, 0])
    assert before == (m.block_table(0), m.block_table(1), m.num_free_blocks())
    m.check_invariants()


def test_reorder_without_room_changes_nothing():
    m = BlockManager(5, 4)
    m.allocate(0, 6)     # blocks 0, 1
    m.allocate(1, 4)     # block 2
    m.allocate(2, 8)     # blocks 3, 4: none is free
    assert m.reorder([0, 1], [0, 1]) == []
    m.fork(1, [3])
    with pytest.raises(OutOfBlocks):
        m.reorder([0, 1], [0, 0])  # block 2 is still sequence 3's
    m.check_invariants()
    assert m.block_table(1) == [2] and m.seq_len(1) == 4
    m.free(3)
    assert m.reorder([0, 1], [0, 0]) == [(1, 2, 2)]  # its own block takes the copy
    m.check_invariants()
    assert m.block_table(1) == [0, 2] and m.num_shared_blocks() == 1


def test_reorder_keeps_a_sequence_that_goes_on_where_it_is():
    m = BlockManager(20, 4)
    m.allocate(0, 6)
    m.fork(0, [1, 2])
    heard = []
    m.add_table_listener(lambda s, first: heard.append((s, first)))
    t1 = m.block_table(1)
    copies = m.reorder([0, 1, 2], [1, 1, 1])
    assert m.block_table(1) == t1 and [c[0] for c in copies] == [t1[1]] * 2 and all(c[2] == 2 for c in copies)
    assert [s for s, _ in heard] == [0, 2] and all(first == 1 for _, first in heard)
    assert m.reorder([0, 1, 2], [1, 0, 2]) == []  # exchanged: nothing to copy
    m.check_invariants()


def test_reorder_between_sequences_of_different_lengths():
    m = BlockManager(20, 4)
    m.allocate(0, 3)
    m.allocate(1, 11)
    copies = m.reorder([0, 1], [1, 1])
    assert m.seq_len(0) == 11 and len(copies) == 1 and copies[0][2] == 3
    m.check_invariants()
    m.allocate(2, 1)
    m.reorder([0, 2], [1, 1])  # the longer one gives its blocks back
    assert m.seq_len(0) == 1
    m.check_invariants()


@pytest.mark.parametrize("seed", range(6))
def test_every_sequence_reads_its_own_history(seed):
    """Random allocations, appends, forks, reorders, truncations and frees over a store of tokens: each sequence's slots hold
    what was appended to it or to the one it comes from."""
    r, B = random.Random(seed), random.Random(seed).choice([1, 3, 4, 16])
    m, store, want, fresh = BlockManager(60, B), {}, {}, iter(range(10 ** 6))

    def make(copies):
        assert len({d for _, d, _ in copies}) == len(copies) and not {s for s, _, _ in copies} & {d for _, d, _ in copies}
        for s, d, n in copies:
            for i in range(n):
                store[d * B + i] = store[s * B + i]

    for _ in range(300):
        op, ids = r.randrange(7), sorted(want)
        try:
            if op == 0 or not ids:
                s, n = next(fresh), r.randrange(3 * B)
                slots = m.allocate(s, n)
                want[s] = [next(fresh) for _ in range(n)]
                store.update(zip(slots, want[s]))
            elif op in (1, 2):
                s, n = r.choice(ids), r.randint(1, B + 1)
                slots = m.append_slots(s, n)
                m.check_own(s, m.seq_len(s) - n, n)
                new = [next(fresh) for _ in range(n)]
                store.update(zip(slots, new))
                want[s] = want[s] + new
            elif op == 3:
                s, new = r.choice(ids), [next(fresh) for _ in range(r.randint(1, 3))]
                make(m.fork(s, new))
                want.update({i: want[s] for i in new})
            elif op == 4:
                some = r.sample(ids, r.randint(1, len(ids)))
                parents = [r.randrange(len(some)) for _ in some]
                make(m.reorder(some, parents))
                want.update(zip(some, [want[some[p]] for p in parents]))
            elif op == 5:
                s = r.choice(ids)
                n = r.randint(0, len(want[s]))
                m.truncate(s, n)
                want[s] = want[s][:n]
            elif len(ids) > 3:
                s = r.choice(ids)
                m.free(s)
                del want[s]
        except OutOfBlocks:
            m.free(ids[0])
            del want[ids[0]]
        except ValueError:
            assert op == 5  # inside a block that others hold
        m.check_invariants()
        for s, tokens in want.items():
            assert [store[x] for x in m.slots(s, 0, m.seq_len(s))] == tokens


def test_writes_and_truncations_inside_shared_blocks_are_refused():
    m = BlockManager(20, 4)
    m.allocate(0, 9)
    m.fork(0, [1])
    with pytest.raises(ValueError, match="sequences hold"):
        build_metadata(m, [(0, 7, 1)], "cpu")
    with pytest.raises(ValueError, match="sequences hold"):
        build_metadata(m, [(1, 3, 6)], "cpu")
    with pytest.raises(ValueError, match="sequences hold"):
        build_tree_metadata(m, [(1, 7, [-1, 0])], "cpu")
    build_metadata(m, [(0, 8, 1), (1, 8, 1)], "cpu")
    with pytest.raises(ValueError, match="sequences hold"):
        m.truncate(1, 7)
    m.truncate(1, 4)
    assert m.append_slots(1, 1)[0] // 4 not in m.block_table(0)
    m.check_invariants()


def test_shared_groups():
    def t(*x):
        return np.asarray(x, dtype=np.int32)

    assert shared_groups([t(1, 2), t(3), t(4, 5)], [8, 4, 8], 4) == []
    # full blocks inside every context
    assert shared_groups([t(1, 2, 3), t(9), t(1, 2, 4)], [9, 4, 11], 4) == [([0, 2], 8)]
    assert shared_groups([t(1, 2, 3), t(1, 2, 4)], [9, 6], 4) == [([0, 1], 4)]
    assert shared_groups([t(1), t(1)], [3, 3], 4) == []
    # two prompts of 20 blocks behind one of 2: two groups read fewer tokens than one
    a, b = list(range(10, 30)), list(range(40, 60))
    tables = [t(1, 2, *a), t(1, 2, *b), t(1, 2, *a, 5), t(1, 2, *b, 6)]
    assert shared_groups(tables, [88, 88, 89, 89], 4) == [([0, 2], 88), ([1, 3], 88)]
    # one that shares little more with another: one group of all
    tables = [t(*range(20), 30), t(*range(20), 30), t(*range(20), 31)]
    assert shared_groups(tables, [84] * 3, 4) == [([0, 1, 2], 80)]


def test_shared_groups_of_a_long_chain():
    """Row i shares i blocks with the rows behind it: groups within groups, more than Python's stack holds."""
    n = 1500
    tables = [np.concatenate([np.arange(i), [10 ** 6 + i]]).astype(np.int32) for i in range(1, n + 1)]
    found = shared_groups(tables, [4 * len(t) for t in tables], 4)
    rows = [r for g, _ in found for r in g]
    assert len(rows) == len(set(rows)) and found
    for g, tokens in found:
        assert tokens % 4 == 0 and all((tables[r][:tokens // 4] == tables[g[0]][:tokens // 4]).all() for r in g)


def test_metadata_names_the_groups_of_decode_rows():
    m = BlockManager(40, 4)
    m.allocate(0, 9)
    m.fork(0, [1, 2])
    m.allocate(7, 5)
    meta = build_metadata(m, [(1, 8, 1), (7, 0, 5), (2, 8, 1), (0, 8, 1)], "cpu")
    assert meta.shared == [([0, 2, 3], 8)]
    tree = build_tree_metadata(m, [(1, 8, [-1])], "cpu")
    assert tree.shared == []
    for s in (1, 2):
        m.free(s)
    assert build_metadata(m, [(0, 8, 1)], "cpu").shared == []


@pytest.mark.parametrize("copies", [[(0, 1)], [(0, 6, 1)], [(-1, 2, 1)], [(0, 1, 5)], [(0, 1, -1)], [(0, 1, 1), (2, 1, 1)],
                                    [(0, 1, 1), (1, 2, 1)], [(3, 3, 2)]])
def test_copy_blocks_refuses(copies):
    k = torch.zeros(2, 1, 6, 4, 8)
    with pytest.raises(ValueError):
        copy_blocks((k, k.clone()), copies)


def test_copy_blocks_refuses_pools():
    k = torch.zeros(2, 1, 6, 4, 8)
    for pools in ((), (k,) * 5, (k, torch.zeros(2, 1, 5, 4, 8)), (k[..., ::2],), (k[0, 0],)):
        with pytest.raises(ValueError):
            copy_blocks(pools, [(0, 1, 1)])
    copy_blocks((k,), [])


def test_copy_blocks_on_the_cpu():
    g = torch.Generator().manual_seed(0)
    pools = [torch.randn(3, 2, 9, 4, 8, generator=g), torch.randn(3, 2, 9, 4, generator=g)]
    want = [t.clone() for t in pools]
    copies = [(0, 3, 2), (0, 4, 4), (7, 8, 0)]
    for t in want:
        t[:, :, 3, :2], t[:, :, 4] = t[:, :, 0, :2], t[:, :, 0]
    copy_blocks(pools, copies)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def _cache(fmt, m):
    if fmt == "bf16":
        return PagedKVCache(CFG, m.num_blocks, m.block_size, "cpu", torch.float64, "gather")
    return QuantPagedKVCache(CFG, m.num_blocks, m.block_size, "cpu", torch.float64, "gather", fmt=fmt, manager=m, n_stage=24)


def _step(model, cache, m, ids, tokens):
    for s in ids:
        m.append_slot(s)
    meta = build_metadata(m, [(s, m.seq_len(s) - 1, 1) for s in ids], "cpu")
    return model.forward(torch.tensor(tokens), meta.positions, cache, meta)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "int8-kchannel"])
@pytest.mark.parametrize("prompt", [4, 7, 16])
def test_beam_search_over_shared_blocks(fmt, prompt):
    """Four beams of two requests, some steps: the logits and the cached K and V are those of sequences that share nothing,
    each of which runs its whole history again (prompt, then token by token, as the beams did). In 64 bits, where the sums'
    orders move no quantized code: 1e-9 is far over what they differ by and far under a code's step."""
    torch.manual_seed(0)
    B, K, steps = 4, 4, 9
    model = Qwen2Model(CFG, "cpu", torch.float64, seed=3, max_positions=64, std=0.3)
    m = BlockManager(80, B)
    cache = _cache(fmt, m)
    r = random.Random(1)
    prompts = [[r.randrange(37) for _ in range(prompt)], [r.randrange(37) for _ in range(prompt + 1)]]
    logits = []
    for i, p in enumerate(prompts):
        m.allocate(10 * i, len(p))
        meta = build_metadata(m, [(10 * i, 0, len(p))], "cpu")
        logits.append(model.forward(torch.tensor(p), meta.positions, cache, meta))
    choice = beam_select(torch.cat(logits).float(), torch.zeros(2), 1, K)
    ids, copies = [], []
    for i in range(2):
        new = [10 * i + j for j in range(1, K)]
        copies += m.fork(10 * i, new)
        ids += [10 * i, *new]
    cache.copy_blocks(copies)
    scores, tokens = choice.scores.reshape(-1), choice.tokens.reshape(-1).tolist()
    texts = [[t] for t in tokens]
    moved = 0
    for _ in range(steps):
        out = _step(model, cache, m, ids, tokens)
        for row, (s, text) in enumerate(zip(ids, texts)):  # alone, in a cache of its own
            m1 = BlockManager(20, B)
            c1 = _cache(fmt, m1)
            p = prompts[row // K]
            m1.allocate(0, len(p))
            meta = build_metadata(m1, [(0, 0, len(p))], "cpu")
            model.forward(torch.tensor(p), meta.positions, c1, meta)
            for t in text:
                want = _step(model, c1, m1, [0], [t])
            assert torch.allclose(out[row], want[0], rtol=1e-9, atol=1e-9)
            for layer in range(2):
                for a, b in zip(cache.gather(layer, row), c1.gather(layer, 0)):
                    assert torch.allclose(a, b, rtol=1e-9, atol=1e-9)
        choice = beam_select(out.float(), scores, K, K)
        parents = (choice.beams + torch.arange(2)[:, None] * K).reshape(-1).tolist()
        moved += sum(p != i for i, p in enumerate(parents))
        cache.copy_blocks(m.reorder(ids, parents))
        m.check_invariants()
        scores, tokens = choice.scores.reshape(-1), choice.tokens.reshape(-1).tolist()
        texts = [texts[p] + [t] for p, t in zip(parents, tokens)]
    assert moved > steps  # the beams did change places
    for s in ids:
        m.free(s)
    assert m.num_free_blocks() == 80
    if fmt == "int8-kchannel":
        assert not cache._stage_of
