"""The C entry points of shared prefixes, beams and copies of blocks refuse bad arguments before any launch, on the CPU."""

import ctypes

import numpy as np
import pytest
import torch

from engine import _hip
from engine.hip_prefix import MAX_CONTEXT, prefix_supported

GOOD = dict(num_seqs=4, num_q_heads=14, num_kv_heads=2, head_dim=64, block_size=16, num_blocks=9, max_context=200, kv_mode=0,
            scale=1.0)


def plan(groups, room=None, over=(), lens=None):
    """(return code, layout, plan) of sipa_prefix_plan."""
    p = _hip.PrefixParams(struct_size=ctypes.sizeof(_hip.PrefixParams), **{**GOOD, **dict(over)})
    starts = np.cumsum([0] + [len(r) for r, _ in groups]).astype(np.int32)
    members = np.asarray([x for r, _ in groups for x in r], dtype=np.int32)
    tokens = np.asarray([t for _, t in groups], dtype=np.int32)
    lens = None if lens is None else np.asarray(lens, dtype=np.int32)
    args = (ctypes.byref(p), len(groups), starts.ctypes.data, members.ctypes.data, tokens.ctypes.data,
            None if lens is None else lens.ctypes.data)
    layout = _hip.PrefixLayout()
    rc = _hip.lib().sipa_prefix_plan(*args, None, 0, ctypes.byref(layout))
    if rc:
        return rc, layout, None
    out = np.full(layout.plan_ints + 1, 77, dtype=np.int32)
    rc = _hip.lib().sipa_prefix_plan(*args, out.ctypes.data, layout.plan_ints if room is None else room, ctypes.byref(layout))
    assert out[-1] == 77
    return rc, layout, out[:-1]


@pytest.mark.parametrize("over", [dict(head_dim=32), dict(block_size=8), dict(num_q_heads=13), dict(num_q_heads=34), dict(kv_mode=2),
                                  dict(max_context=0), dict(max_context=(1 << 24) + 1), dict(num_seqs=-1), dict(num_kv_heads=0)])
def test_plans_refuse_sizes(over):
    assert plan([], over=over)[0] in (_hip.EINVAL, _hip.EUNSUPPORTED)


@pytest.mark.parametrize("groups", [[([0, 1], 15)], [([0, 1], -16)], [([0, 1], 208)], [([0, 4], 16)], [([-1, 0], 16)],
                                    [([0, 0], 16)], [([0, 1], 16), ([1, 2], 16)], [([0, 1, 2, 3, 0], 16)]])
def test_plans_refuse_groups(groups):
    assert plan(groups)[0] == _hip.EINVAL


def test_plans_refuse_too_little_room():
    assert plan([([0, 1], 16)], room=10)[0] == _hip.EINVAL


@pytest.mark.parametrize("lens", [None, [200, 199, 65, 1], [0, 0, 0, 0], [10, 64, 64, 200], [-5, 900, 64, 3]])
@pytest.mark.parametrize("groups", [[], [([0, 1, 2], 64)], [([3, 1], 192), ([0, 2], 16)], [([2], 64), ([], 0), ([0, 1], 0)]])
def test_plans_cover_every_key_once(groups, lens):
    """Items: each group's rows and shared keys, once a KV head; pieces: as many as each row has been given; states apart."""
    rc, l, p = plan(groups, lens=lens)
    assert rc == 0 and l.plan_ints == p.size
    items = p[:8 * l.num_items].reshape(-1, 8)
    pieces = p[8 * l.num_items:8 * (l.num_items + l.num_pieces)].reshape(-1, 8)
    rows = p[8 * (l.num_items + l.num_pieces):][:32].reshape(-1, 8)
    members = p[8 * (l.num_items + l.num_pieces + 4):]
    assert members.tolist() == [x for r, _ in groups for x in r]
    assert sorted(items[:, 7]) == list(range(l.num_items)) and pieces[:, 5].tolist() == list(range(l.num_pieces))
    seen = set()
    for table_row, first, M, m0, h, lo, hi, _ in items.tolist():
        g = next(r for r, t in groups if len(r) > 1 and t and table_row in r)
        assert M == len(g) * 7 and members[first] == table_row and lo % 64 == 0
        for key in range(lo, hi):
            for m in range(m0, min(m0 + l.tile_rows, M)):
                assert (table_row, h, m, key) not in seen
                seen.add((table_row, h, m, key))
    assert len(seen) == sum(2 * 7 * len(r) * t for r, t in groups if len(r) > 1)
    for s in range(4):
        mine = [(h, i) for x, h, i, *_ in pieces.tolist() if x == s]
        assert mine == [(h, i) for h in range(2) for i in range(rows[s, 6])] and pieces[rows[s, 5], 0] == s


def test_the_predicate_is_the_librarys():
    for d in (32, 64, 128):
        for b in (8, 16, 32, 64):
            for g in (1, 16, 17):
                for c in (1, MAX_CONTEXT, MAX_CONTEXT + 1):
                    rc, *_ = plan([], over=dict(head_dim=d, block_size=b, num_q_heads=2 * g, max_context=c, num_seqs=1))
                    assert (rc == 0) == prefix_supported(torch.bfloat16, torch.int8, b, d, g, c)
    assert not prefix_supported(torch.float32, torch.float32, 16, 64, 1)


def test_attention_refuses():
    p = _hip.PrefixParams(struct_size=ctypes.sizeof(_hip.PrefixParams), **GOOD)
    call = _hip.lib().sipa_prefix_attention
    assert call(ctypes.byref(p), None) == _hip.EINVAL  # no block tables
    p.bt_width = 13
    assert call(ctypes.byref(p), None) == _hip.EINVAL  # no tensors
    p.q = p.k_cache = p.v_cache = p.block_tables = p.context_lens = p.out = p.plan = 4096
    assert call(ctypes.byref(p), None) == _hip.EINVAL  # no layout
    p.layout.tile_rows, p.layout.num_pieces = 64, 8
    assert call(ctypes.byref(p), None) == _hip.EWORKSPACE
    p.layout.num_pieces = 7
    assert call(ctypes.byref(p), None) == _hip.EINVAL
    p.layout.num_pieces, p.q = 8, 4098
    assert call(ctypes.byref(p), None) == _hip.EINVAL
    p.num_seqs = 0
    assert call(ctypes.byref(p), None) == 0
    p.struct_size -= 8
    assert call(ctypes.byref(p), None) == _hip.EINVAL


def test_selection_refuses():
    good = dict(num_rows=8, vocab=100, num_groups=2, beams=4, num_candidates=8, dtype=1, logits=4096, logits_stride=100, scores=4096,
                out_scores=4096, out_beams=4096, out_tokens=4096)

    def call(**over):
        p = _hip.BeamParams(struct_size=ctypes.sizeof(_hip.BeamParams), **{**good, **over})
        return _hip.lib().sipa_beam_select(ctypes.byref(p), None)

    assert call() == _hip.EWORKSPACE
    for over in (dict(num_candidates=0), dict(num_candidates=65), dict(vocab=0), dict(vocab=(1 << 25) + 1), dict(dtype=3),
                 dict(beams=5), dict(beams=0), dict(num_rows=-1), dict(logits=None), dict(out_beams=None), dict(beams=1025)):
        assert call(**over) in (_hip.EINVAL, _hip.EUNSUPPORTED), over
    assert call(num_groups=0) == 0


def test_copies_are_checked():
    def check(copies):
        flat = np.asarray(copies, dtype=np.int32)
        return _hip.lib().sipa_check_copies(flat.ctypes.data, len(copies), 5000, 16)

    many = [(i, 2500 + i, 16) for i in range(2500)]
    assert check([(0, 1, 16)]) == check(many) == check([(0, 1, 1), (0, 2, 1), (4999, 3, 0)]) == 0
    for bad in ([(0, 0, 1)], [(0, 5000, 1)], [(-1, 0, 1)], [(0, 1, 17)], [(0, 1, 1), (1, 2, 1)], [(0, 1, 1), (3, 1, 1)],
                many + [(7, 2600, 1)], many + [(2700, 2499, 1)]):
        assert check(bad) == _hip.EINVAL, bad[-1]
    p = _hip.CopyParams(struct_size=ctypes.sizeof(_hip.CopyParams), num_layers=1, num_kv_heads=1, num_blocks=9, block_size=256,
                        num_pools=1, num_copies=1)
    assert _hip.lib().sipa_copy_blocks(ctypes.byref(p), None) == _hip.EUNSUPPORTED
    p.block_size = 16
    assert _hip.lib().sipa_copy_blocks(ctypes.byref(p), None) == _hip.EINVAL
    p.num_pools = 5
    assert _hip.lib().sipa_copy_blocks(ctypes.byref(p), None) == _hip.EINVAL
    p.num_pools, p.num_copies = 1, 0
    assert _hip.lib().sipa_copy_blocks(ctypes.byref(p), None) == 0
