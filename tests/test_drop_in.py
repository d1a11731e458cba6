"""The caches' modules beside the reference's own block manager, config, attention and quantizer: what has to be copied for them
to import, and that they serve a manager with the reference's interface alone (engine/block_manager.py:19-137). CPU."""

import ast
import os
import shutil
import subprocess
import sys
from pathlib import Path

from engine import _hip

ENGINE = Path(_hip.__file__).parent
COPIED = {"_hip", "hip_beam", "hip_decode", "hip_prefill", "hip_prefix", "hip_quant", "hip_tree", "paged_cache", "quant_cache"}
THEIRS = {"attention", "block_manager", "config", "quant"}

MANAGER = '''
class BlockManager:
    """Blocks handed out in order; the reference's names."""

    def __init__(self, num_blocks, block_size=16):
        self.num_blocks, self.block_size = num_blocks, block_size
        self.free_blocks, self.tables, self.lengths, self.listeners = list(range(num_blocks)), {}, {}, []

    def add_free_listener(self, fn):
        self.listeners.append(fn)

    def allocate(self, seq_id, n_tokens):
        self.tables[seq_id], self.lengths[seq_id] = [], 0
        self.append_slots(seq_id, n_tokens)

    def append_slots(self, seq_id, n=1):
        self.lengths[seq_id] += n
        while len(self.tables[seq_id]) * self.block_size < self.lengths[seq_id]:
            self.tables[seq_id].append(self.free_blocks.pop(0))

    def block_table(self, seq_id):
        return list(self.tables[seq_id])

    def seq_len(self, seq_id):
        return self.lengths[seq_id]

    def free(self, seq_id):
        blocks = self.tables.pop(seq_id)
        self.free_blocks += blocks
        for fn in self.listeners:
            fn(blocks)
'''

PROGRAM = '''
import torch
from engine.block_manager import BlockManager
from engine.config import ModelConfig
from engine.paged_cache import PagedKVCache, build_metadata
from engine.quant_cache import QuantPagedKVCache

cfg = ModelConfig(vocab_size=37, hidden_size=28, intermediate_size=24, num_layers=2, num_q_heads=7, num_kv_heads=1, head_dim=4)
for fmt in ("bf16", "int8", "int8-kchannel"):
    m = BlockManager(20, 4)
    if fmt == "bf16":
        cache = PagedKVCache(cfg, 20, 4, "cpu", torch.float32, "gather")
    else:
        cache = QuantPagedKVCache(cfg, 20, 4, "cpu", torch.float32, "gather", fmt=fmt, manager=m, n_stage=4)
    torch.manual_seed(0)
    m.allocate(0, 6), m.allocate(1, 9)
    for batch in ([(0, 0, 6), (1, 0, 9)], [(0, 6, 1), (1, 9, 1)], [(1, 10, 1)]):
        for s, start, n in batch:
            m.append_slots(s, start + n - m.seq_len(s))
        meta = build_metadata(m, batch, "cpu")
        T = meta.num_tokens
        cache.begin(T, meta)
        for layer in range(2):
            cache.write(layer, torch.randn(T, 1, 4), torch.randn(T, 1, 4))
            out = cache.attend(layer, torch.randn(T, 7, 4), meta.positions, 0.5)
            assert out.shape == (T, 28) and out.isfinite().all()
    m.free(0), m.free(1)
    assert not getattr(cache, "_stage_of", {})
print("served")
'''


def imports(module):
    tree = ast.parse((ENGINE / f"{module}.py").read_text())
    for n in ast.walk(tree):
        if isinstance(n, ast.ImportFrom) and n.level == 1:
            yield from [n.module] if n.module else [a.name for a in n.names]


def test_the_modules_that_the_caches_need():
    todo, seen = ["paged_cache", "quant_cache"], set()
    while todo:
        x = todo.pop()
        if x not in seen:
            seen.add(x)
            todo += [] if x in THEIRS else imports(x)
    assert seen == COPIED | THEIRS


def test_caches_over_a_manager_with_the_references_interface(tmp_path):
    package = tmp_path / "engine"
    package.mkdir()
    (package / "__init__.py").write_text("")
    for name in COPIED | THEIRS - {"block_manager"}:
        shutil.copy(ENGINE / f"{name}.py", package)
    (package / "block_manager.py").write_text(MANAGER)
    env = {**os.environ, "SIPA_LIB": str(_hip.LIB_PATH), "PYTHONPATH": str(tmp_path)}
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=tmp_path, env=env, capture_output=True, text=True, timeout=110)
    assert done.returncode == 0 and done.stdout == "served\n", done.stderr[-2000:]
