"""Which sequences of a forward are searched for groups: those whose tables begin with a shared block. CPU."""

import random

from engine import paged_cache
from engine.block_manager import BlockManager, OutOfBlocks
from engine.hip_prefix import shared_groups
from engine.paged_cache import build_metadata


def searched(monkeypatch):
    seen = []
    monkeypatch.setattr(paged_cache, "shared_groups", lambda tables, lens, B: seen.append(len(tables)) or shared_groups(tables, lens, B))
    return seen


def test_sequences_of_their_own_are_not_searched(monkeypatch):
    seen = searched(monkeypatch)
    m = BlockManager(100, 4)
    for s in range(8):
        m.allocate(s, 9)
    batch = [(s, 8, 1) for s in range(8)]
    assert build_metadata(m, batch, "cpu").shared == [] and seen == []
    m.fork(7, [20])  # one that is not in the batch
    assert build_metadata(m, batch, "cpu").shared == [] and seen == []
    m.fork(3, [21])
    meta = build_metadata(m, [*batch, (21, 8, 1)], "cpu")
    assert meta.shared == [([3, 8], 8)] and seen == [3]  # 3, 7 and 21


def test_groups_are_those_of_all_sequences():
    """Over random forks, reorders, truncations and frees: as if every sequence were searched."""
    r, m, fresh = random.Random(1), BlockManager(200, 4), iter(range(10 ** 6))
    found = 0
    for _ in range(400):
        ids = m.seq_ids()
        try:
            op = r.randrange(6)
            if op == 0 or not ids:
                m.allocate(next(fresh), r.randint(1, 30))
            elif op == 1:
                m.append_slots(r.choice(ids), r.randint(1, 6))
            elif op == 2:
                m.fork(r.choice(ids), [next(fresh) for _ in range(r.randint(1, 3))])
            elif op == 3:
                some = r.sample(ids, r.randint(1, len(ids)))
                m.reorder(some, [r.randrange(len(some)) for _ in some])
            elif op == 4:
                s = r.choice(ids)
                m.truncate(s, m.seq_len(s) // 4 * r.randint(1, 4))
            elif len(ids) > 5:
                m.free(r.choice(ids))
        except OutOfBlocks:
            for s in ids[:3]:
                m.free(s)
        except ValueError:
            assert op == 4  # a truncation inside a shared block
        live = [s for s in m.seq_ids() if m.seq_len(s) > 0]
        tables, lens = [m.table_array(s) for s in live], [m.seq_len(s) for s in live]
        want = shared_groups(tables, lens, 4) if m.num_shared_blocks() else []
        got = paged_cache.decode_groups(m, tables, lens, [1] * len(live))
        assert got == want
        found += len(got)
    assert found > 100
