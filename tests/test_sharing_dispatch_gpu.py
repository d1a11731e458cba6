"""Forwards over forked sequences that the shared-prefix kernel cannot take as they come: each is answered, as it is where the
sequences share nothing."""

import pytest
import torch

from engine.block_manager import BlockManager
from engine.config import ModelConfig
from engine.hip_decode import DecodePlan
from engine.hip_prefix import PrefixPlan
from engine.paged_cache import PagedKVCache, build_metadata
from engine.quant_cache import QuantPagedKVCache

pytestmark = pytest.mark.gpu
CFG = ModelConfig(vocab_size=64, hidden_size=448, intermediate_size=64, num_layers=2, num_q_heads=7, num_kv_heads=1, head_dim=64)


def forked(fmt="bf16", members=4, tokens=700):
    """A cache that takes the shared-prefix kernel however little is shared, and the metadata of a step over forked sequences."""
    m = BlockManager(60 + members, 16)
    if fmt == "bf16":
        cache = PagedKVCache(CFG, m.num_blocks, 16, "cuda", torch.bfloat16, "hip")
        cache.k.normal_(), cache.v.normal_()
    else:
        cache = QuantPagedKVCache(CFG, m.num_blocks, 16, "cuda", torch.bfloat16, "hip", fmt=fmt, manager=m)
        for t in (cache.k, cache.v):
            t.copy_(torch.randint(-127, 128, t.shape, device="cuda"))
        for t in (cache.k_scale, cache.v_scale):
            t.uniform_(0.005, 0.02)
    cache.prefix_min_bytes = 1
    m.allocate(0, tokens)
    m.fork(0, list(range(1, members)))
    for s in range(members):
        m.append_slot(s)
    meta = build_metadata(m, [(s, tokens, 1) for s in range(members)], "cuda")
    assert meta.shared
    return cache, meta


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_captured_forwards_go_to_the_decode_kernel(fmt):
    cache, meta = forked(fmt)
    q = [torch.randn(4, 7, 64, device="cuda").bfloat16() for _ in range(2)]

    def step():
        cache.begin(4, meta)
        return [cache.attend(layer, q[layer], meta.positions, 0.125) for layer in range(2)]

    shared = meta.shared
    step()
    assert type(cache._plan) is PrefixPlan
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    assert type(cache._plan) is DecodePlan
    for _ in range(4):
        for x in q:
            x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        meta.shared = []
        want = step()
        assert type(cache._plan) is DecodePlan and all(torch.equal(a, b) for a, b in zip(out, want))
        meta.shared = shared
        eager = step()
        assert type(cache._plan) is PrefixPlan
        # each kernel: 2^-8 of the result (its rounding), and under 2^-12 of the weights' sum of |v| (scores, exponentials, two
        # bf16 terms of the weights), which is at most the largest |v|, under 8
        for a, b in zip(eager, want):
            assert ((a.double() - b.double()).abs() <= 2 ** -7 * b.double().abs() + 2 * 2 ** -12 * 8).all()


@pytest.mark.parametrize("rows", ["head stride", "row stride", "address"])
def test_rows_at_any_alignment(rows):
    """q that the decode kernels take although no 16-byte load fits it: the first layer's, or a later one's alone."""
    cache, meta = forked()
    q = torch.randn(4, 7, 64, device="cuda").bfloat16()
    odd = {"head stride": lambda: torch.empty(4, 7, 65, device="cuda", dtype=torch.bfloat16)[..., :64],
           "row stride": lambda: torch.empty(4, 7 * 64 + 1, device="cuda", dtype=torch.bfloat16)[:, :448].view(4, 7, 64),
           "address": lambda: torch.empty(4 * 448 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(4, 7, 64)}[rows]().copy_(q)
    cache.begin(4, meta)
    want = [cache.attend(layer, q, meta.positions, 0.125) for layer in range(2)]
    for first, second in ((odd, odd), (q, odd), (odd, q)):
        cache.begin(4, meta)
        got = [cache.attend(layer, x, meta.positions, 0.125) for layer, x in enumerate((first, second))]
        assert type(cache._plan) is PrefixPlan and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("fmt,head_dim,rows,kernel", [("int8", 64, 311, DecodePlan), ("int8", 64, 312, PrefixPlan), ("int8", 128, 48, DecodePlan),
                                                      ("int8", 128, 49, PrefixPlan), ("bf16", 64, 48, DecodePlan), ("bf16", 64, 49, PrefixPlan)])
def test_what_a_cache_takes_the_kernel_for(fmt, head_dim, rows, kernel):
    """A cache's own limits, for one KV head and 4096 shared tokens: INT8 at head_dim 64 from 160 MiB that would be read again
    (310.3 times 4096 tokens of 132 bytes), at 128 from 48 MiB (47.3 times, 260 bytes), bf16 from 48 MiB (48 times, 256 bytes)."""
    cfg = ModelConfig(vocab_size=64, hidden_size=448, intermediate_size=64, num_layers=1, num_q_heads=7, num_kv_heads=1, head_dim=head_dim)
    m = BlockManager(256 + rows, 16)
    if fmt == "bf16":
        cache = PagedKVCache(cfg, m.num_blocks, 16, "cuda", torch.bfloat16, "hip")
    else:
        cache = QuantPagedKVCache(cfg, m.num_blocks, 16, "cuda", torch.bfloat16, "hip", fmt=fmt, manager=m)
    cache.k.zero_(), cache.v.zero_()
    m.allocate(0, 4096)
    m.fork(0, list(range(1, rows)))
    for s in range(rows):
        m.append_slot(s)
    meta = build_metadata(m, [(s, 4096, 1) for s in range(rows)], "cuda")
    cache.begin(rows, meta)
    out = cache.attend(0, torch.zeros(rows, 7, head_dim, device="cuda").bfloat16(), meta.positions, 0.125)
    assert type(cache._plan) is kernel and not out.any()
