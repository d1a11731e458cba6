"""The contexts that the tree attention kernel takes: its predicate says what the library refuses, and a forward past it goes
through the gather path."""

import ctypes

import pytest
import torch

from engine import _hip
from engine.block_manager import BlockManager
from engine.config import ModelConfig
from engine.hip_tree import tree_supported
from engine.paged_cache import PagedKVCache, build_tree_metadata


def library_takes(head_dim, group, nodes, context, block, kv_mode):
    p = _hip.TreeParams(struct_size=ctypes.sizeof(_hip.TreeParams), num_seqs=1, num_tokens=nodes, num_q_heads=2 * group,
                        num_kv_heads=2, head_dim=head_dim, block_size=block, num_blocks=8, max_context=context, max_nodes=nodes,
                        words=4, scale=1.0, kv_mode=kv_mode, num_splits=1)
    return _hip.lib().sipa_tree_workspace_bytes(ctypes.byref(p), None) >= 0


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("group,nodes", [(1, 1), (7, 9), (7, 10), (64, 1), (64, 2), (1, 64), (1, 65), (6, 256)])
@pytest.mark.parametrize("pool,kv_mode", [(torch.bfloat16, 0), (torch.int8, 1)])
def test_the_predicate_is_the_librarys(head_dim, group, nodes, pool, kv_mode):
    limits = (1, 655360, 1179648, 2097152)
    for context in (c + d for c in limits for d in (-1, 0, 1)):
        if context < 1:
            continue
        assert tree_supported(torch.bfloat16, pool, 16, head_dim, group, context, nodes) == \
            library_takes(head_dim, group, nodes, context, 16, kv_mode), context
    assert not tree_supported(torch.bfloat16, pool, 16, head_dim, group, 2097153, nodes)
    assert not tree_supported(torch.bfloat16, pool, 16, head_dim, group, 100, 257)


@pytest.mark.gpu
@pytest.mark.parametrize("context", [655360, 655361])
def test_forwards_past_the_limit_take_the_gather_path(context):
    """14 nodes of 7 heads, so more than 64 rows: the kernel to 655360 keys, then the gather path's own result. K and V hold 64
    tokens over and over, so that the rows are also those of 64 keys. Of the sum of p |v| they differ by: 2^-11, each token's
    count being one more or less than the others' beside 10240 (the nodes' masks too); scores rounded to bf16 by the gather
    path, 2^-8 of them, in the numerator and the denominator; probabilities rounded to bf16, 2^-8; n keys added up 16 at a
    time in fp32; and of the result its rounding to bf16, 2^-8."""
    cfg = ModelConfig(vocab_size=16, hidden_size=448, intermediate_size=16, num_layers=1, num_q_heads=7, num_kv_heads=1,
                      head_dim=64)
    m = BlockManager(-(-context // 16) + 2, 16)
    m.allocate(0, context)
    cache = PagedKVCache(cfg, m.num_blocks, 16, "cuda", torch.bfloat16, "hip")
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(4, 16, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    for pool, x in ((cache.k, k), (cache.v, v)):
        pool[0, 0] = x.repeat(-(-m.num_blocks // 4), 1, 1)[:m.num_blocks]
    meta = build_tree_metadata(m, [(0, context - 14, list(range(-1, 13)))], "cuda")
    q = torch.randn(14, 7, 64, generator=g, device="cuda").bfloat16()
    print("context", context, flush=True)
    cache.begin(14, meta)
    got = cache.attend(0, q, meta.positions, 0.125)
    cache.attn_backend = "gather"
    cache.begin(14, meta)
    gather = cache.attend(0, q, meta.positions, 0.125)
    assert torch.equal(got, gather) == (context > 655360)
    z = q.double().cpu().view(98, 64) @ k.double().cpu().view(64, 64).T * 0.125
    p = torch.softmax(z, 1)
    want, size = p @ v.double().cpu().view(64, 64), p @ v.double().cpu().view(64, 64).abs()
    err = (got.double().cpu().view(98, 64) - want).abs()
    eps = 2.0 ** -11 + 2.0 ** -7 * z.abs().amax(1, keepdim=True) + 2.0 ** -8 + context / 16 * 2.0 ** -24
    assert (err <= eps * size + 2.0 ** -8 * want.abs()).all(), (err / size).max()
