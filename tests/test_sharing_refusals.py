"""Steps that would write into blocks that several sequences hold, through the device's block tables and the graph runner."""

import pytest
import torch

from engine.block_manager import BlockManager
from engine.config import ModelConfig
from engine.device_tables import DeviceBlockTables
from engine.graph_runner import DecodeGraphRunner
from engine.model import Qwen2Model
from engine.paged_cache import PagedKVCache, build_metadata
from engine.quant_cache import QuantPagedKVCache

CFG = ModelConfig(vocab_size=211, hidden_size=448, intermediate_size=64, num_layers=2, num_q_heads=7, num_kv_heads=1, head_dim=64)


def test_device_tables_refuse_writes_into_shared_blocks():
    """Refused on the host, before anything is uploaded: on CPU tensors here."""
    m = BlockManager(20, 4)
    tables = DeviceBlockTables(m, "cpu", 4, 8)
    m.allocate(0, 9)
    m.fork(0, [1])
    before = tables.table.clone()
    for batch in ([(0, 7, 1)], [(1, 3, 6)], [(1, 8, 1), (0, 0, 9)]):
        with pytest.raises(ValueError, match="sequences hold"):
            tables.build(batch)
    for batch in ([(1, 7, [-1, 0])], [(0, 8, [-1]), (1, 4, [-1, 0, 0])]):
        with pytest.raises(ValueError, match="sequences hold"):
            tables.build_tree(batch)
    assert torch.equal(tables.table, before)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("fmt", ["bf16", "int8", "int8-kchannel"])
def test_the_runner_refuses_to_write_into_a_shared_block(fmt, graph):
    """Forked at a block's end, a sequence whose newest position is in the shared block cannot be stepped before it has a slot
    of its own: refused with nothing written; the step after it is that of a runner that was never asked."""
    outs = []
    for refused in (False, True):
        m = BlockManager(30, 16)
        if fmt == "bf16":
            cache = PagedKVCache(CFG, 30, 16, "cuda", torch.bfloat16, "hip")
        else:
            cache = QuantPagedKVCache(CFG, 30, 16, "cuda", torch.bfloat16, "hip", fmt=fmt, manager=m, n_stage=8)
        model = Qwen2Model(CFG, "cuda", torch.bfloat16, seed=1, max_positions=128, std=0.05)
        m.allocate(0, 32)
        meta = build_metadata(m, [(0, 0, 32)], "cuda")
        model.forward(torch.arange(32, device="cuda"), meta.positions, cache, meta)
        runner = DecodeGraphRunner(model, cache, m, 2, 64)
        assert m.fork(0, [1]) == []
        tokens = torch.tensor([5, 9], device="cuda")
        if refused:
            runner.capture(2)
            pools = [t.view(torch.uint8).clone() for t in (cache.k, cache.v)]  # bits: what was never written may be NaN
            slots = dict(getattr(cache, "_stage_of", {}))
            for seqs in ([0, 1], [1, 0]):
                with pytest.raises(ValueError, match="sequences hold"):
                    runner.step(seqs, tokens, graph=graph)
            m.append_slot(0)
            with pytest.raises(ValueError, match="sequences hold"):
                runner.step([0, 1], tokens, graph=graph)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(pools, (cache.k, cache.v)))
            assert slots == dict(getattr(cache, "_stage_of", {}))
        else:
            m.append_slot(0)
        m.append_slot(1)
        outs.append(runner.step([0, 1], tokens, graph=graph).clone())
        runner.close()
        m.check_invariants()
    assert torch.equal(*outs) and outs[0].isfinite().all()
