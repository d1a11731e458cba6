"""Truncation where an int8-kchannel cache lives on the manager's blocks: a block whose K is quantized by channel cannot be
kept in part (its bf16 rows are gone), and a truncation that would is refused before anything changes."""

import pytest
import torch

from engine.block_manager import BlockManager
from engine.model import Qwen2Model
from engine.paged_cache import build_metadata
from engine.quant_cache import QuantPagedKVCache
from test_tree_cache import SMALL, close


def start(prompt):
    m = BlockManager(64, 16)
    model = Qwen2Model(SMALL, "cpu", torch.float32, seed=1, max_positions=256, std=0.1)
    cache = QuantPagedKVCache(SMALL, 64, 16, "cpu", torch.float32, "gather", "int8-kchannel", m, n_stage=4)
    m.allocate(0, len(prompt))
    meta = build_metadata(m, [(0, 0, len(prompt))], "cpu")
    model.forward(prompt, meta.positions, cache, meta)
    return m, model, cache


def step(m, model, cache, tokens):
    at = m.seq_len(0)
    m.append_slots(0, len(tokens))
    meta = build_metadata(m, [(0, at, len(tokens))], "cpu")
    return model.forward(tokens, meta.positions, cache, meta)


def test_a_quantized_block_is_not_kept_in_part():
    m, model, cache = start(torch.arange(40) % 90)
    table, free = m.block_table(0), m.num_free_blocks()
    for keep in (1, 15, 17, 31):
        with pytest.raises(ValueError, match="block"):
            m.truncate(0, keep)
    assert m.block_table(0) == table and m.seq_len(0) == 40 and m.num_free_blocks() == free
    m.check_invariants()


@pytest.mark.parametrize("keep", [40, 39, 33, 32, 16, 0])
def test_staged_tokens_and_whole_blocks_are(keep):
    """The sequence goes on as one that never held the tokens given up."""
    prompt, more = torch.arange(40) % 90, torch.arange(50, 57)
    m, model, cache = start(prompt)
    m.truncate(0, keep)
    m.check_invariants()
    got = step(m, model, cache, more)
    o, omodel, ocache = start(prompt[:keep]) if keep else (BlockManager(64, 16), model, None)
    if not keep:
        ocache = QuantPagedKVCache(SMALL, 64, 16, "cpu", torch.float32, "gather", "int8-kchannel", o, n_stage=4)
        o.allocate(0, 0)
    want = step(o, omodel, ocache, more)
    close(got, want, 0.02, 5e-3, "after the truncation")  # 8-bit codes of K and V of two chunks of other lengths


def test_other_caches_truncate_anywhere():
    m = BlockManager(64, 16)
    QuantPagedKVCache(SMALL, 64, 16, "cpu", torch.float32, "gather", "int8", m)
    m.allocate(0, 40)
    m.truncate(0, 17)
    assert m.seq_len(0) == 17
