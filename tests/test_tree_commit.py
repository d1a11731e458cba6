"""Commits after a forward over drafted trees keep paths only: a node's K is rotated for its place in the tree, so one that
moves to another place would leave a cache that no sequence of tokens has."""

import pytest
import torch

from engine.paged_cache import build_tree_metadata
from test_tree_cache import prefill, setup

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
PARENTS = [[-1, 0, 1, 0, 3, -1, 5], [-1, -1, 0]]


def after_a_forward(device, fmt="bf16"):
    cfg, m, model, cache = setup(device, fmt)
    prompts = [torch.arange(3, 3 + n, device=device) for n in (20, 9)]
    prefill(model, cache, m, prompts, device)
    for s, p in enumerate(PARENTS):
        m.append_slots(s, len(p))
    meta = build_tree_metadata(m, [(s, len(prompts[s]), p) for s, p in enumerate(PARENTS)], device)
    model.forward(torch.arange(10, device=device), meta.positions, cache, meta)
    return cache, meta


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("accepted", [
    [[0, 2], []],  # node 2 is a child of 1
    [[0, 1, 3], []],  # 3 is 1's sibling
    [[1], []],  # not from a root
    [[0, 5], []],  # two roots
    [[0, 1, 2], [0, 1]],  # the second sequence's
    [[0, 1, 2], [1, 2]],
])
def test_sets_that_are_no_path_are_refused(device, accepted):
    cache, meta = after_a_forward(device)
    before = cache.k.clone(), cache.v.clone()  # places that were never written may hold NaN: the bits are compared
    for given in (None, meta):
        with pytest.raises(ValueError, match="path"):
            cache.commit(accepted, given)
    for a, b in zip((cache.k, cache.v), before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_paths_are_kept(device, fmt):
    for accepted in ([[0, 3, 4], [0, 2]], [[5, 6], [1]], [[], [0]], [[0], []]):
        cache, meta = after_a_forward(device, fmt)
        k, B = cache.k.clone(), cache.block_size
        cache.commit(accepted)
        for i, (start, path) in enumerate(zip(meta.starts(), accepted)):
            table = meta.block_ids_cpu[i]
            for j, node in enumerate(path):
                to, frm = start + j, start + node
                assert torch.equal(cache.k[:, :, table[to // B], to % B], k[:, :, table[frm // B], frm % B])
