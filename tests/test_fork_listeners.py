"""A fork that a table listener refuses leaves the manager, its listeners and the pool as they were. CPU."""

import pytest

from engine.block_manager import BlockManager
from engine.device_tables import DeviceBlockTables


def state(m):
    return {s: (m.block_table(s), m.seq_len(s)) for s in m.seq_ids()}, m.num_free_blocks(), m.num_shared_blocks()


@pytest.mark.parametrize("tokens", [0, 6, 8])
@pytest.mark.parametrize("rows", [1, 2, 3])
def test_forks_past_the_device_tables_rows(tokens, rows):
    m = BlockManager(20, 4)
    larger, tables = DeviceBlockTables(m, "cpu", 8, 8), DeviceBlockTables(m, "cpu", rows, 8)
    freed = []
    m.add_free_listener(freed.extend)
    m.allocate(0, tokens)
    before = state(m)
    with pytest.raises(RuntimeError, match="live sequences"):
        m.fork(0, [1, 2, 3])
    assert state(m) == before
    m.check_invariants()
    # what each listener heard of has been taken back too: there is room for as many sequences as before
    for t, n in ((larger, 8), (tables, rows)):
        assert len(t._free_rows) == n - 1 and set(t._row_of) == set(t._dirty) == {0}
    assert not set(freed) & set(m.block_table(0))
    if rows > 1:
        copies = m.fork(0, list(range(1, rows)))
        assert len(copies) == (rows - 1 if tokens % 4 else 0)
        assert [d for _, d, _ in copies] == list(range(-(-tokens // 4), -(-tokens // 4) + len(copies)))  # the stack's order
    for s in m.seq_ids():
        m.free(s)
    assert m.num_free_blocks() == 20
    m.check_invariants()
