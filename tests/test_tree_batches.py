"""Batches of drafted trees: each sequence once, as two trees of one would take the same slots."""

import pytest
import torch

from engine.block_manager import BlockManager
from engine.device_tables import DeviceBlockTables
from engine.paged_cache import build_tree_metadata

BATCHES = [[(0, 20, [-1, 0]), (0, 20, [-1])], [(0, 20, [-1, 0]), (1, 4, [-1]), (0, 22, [-1])]]


def manager():
    m = BlockManager(16, 16)
    m.allocate(0, 25), m.allocate(1, 5)
    return m


@pytest.mark.parametrize("batch", BATCHES)
def test_a_sequence_twice_is_refused(batch):
    m = manager()
    with pytest.raises(ValueError, match="twice"):
        build_tree_metadata(m, batch, "cpu")
    build_tree_metadata(m, batch[:1] + [(1, 4, [-1])], "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("batch", BATCHES)
def test_a_sequence_twice_is_refused_on_the_device(batch):
    m = manager()
    tables = DeviceBlockTables(m, "cuda", max_seqs=4, max_blocks=8)
    with pytest.raises(ValueError, match="twice"):
        tables.build_tree(batch)
    assert torch.equal(tables.build_tree(batch[:1]).slot_mapping, build_tree_metadata(m, batch[:1], "cuda").slot_mapping)
