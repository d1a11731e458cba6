"""The entry points of drafted trees and of the rules on logits refuse bad arguments on the host, before anything is launched
(no GPU needed). Pointers are made up: a call that got past its checks would fail at its launch with another code."""

import ctypes

import pytest

from engine import _hip

PTR = 1 << 20  # aligned to all that is asked for


def filled(cls, **values):
    p = cls()
    p.struct_size = ctypes.sizeof(cls)
    for name, kind in cls._fields_:
        if kind is ctypes.c_void_p:
            setattr(p, name, PTR)
    for k, v in values.items():
        setattr(p, k, v)
    return p


def tree(**over):
    base = dict(num_seqs=2, num_tokens=8, num_q_heads=14, num_kv_heads=2, head_dim=64, block_size=16, num_blocks=64, max_context=100,
                max_nodes=4, words=1, scale=0.125, q_stride_t=14 * 64, q_stride_h=64, out_stride_t=14 * 64, out_stride_h=64,
                kv_stride_h=64 * 16 * 64, kv_stride_n=16 * 64, bt_stride_s=8, bt_width=8, num_splits=1, workspace_bytes=0,
                k_scale_dtype=_hip.F16, v_scale_dtype=_hip.F16)
    return filled(_hip.TreeParams, **{**base, **over})


@pytest.mark.parametrize("over,code", [
    ({"struct_size": 8}, _hip.EINVAL),
    ({"num_seqs": -1}, _hip.EINVAL),
    ({"num_q_heads": 13}, _hip.EINVAL),
    ({"num_q_heads": 130}, _hip.EUNSUPPORTED),  # group 65
    ({"head_dim": 96}, _hip.EUNSUPPORTED),
    ({"block_size": 8}, _hip.EUNSUPPORTED),
    ({"max_context": 0}, _hip.EUNSUPPORTED),
    ({"max_nodes": 0}, _hip.EUNSUPPORTED),
    ({"max_nodes": 257, "words": 4}, _hip.EUNSUPPORTED),
    ({"max_nodes": 65}, _hip.EINVAL),  # one word
    ({"words": 5}, _hip.EINVAL),
    ({"kv_mode": 2}, _hip.EUNSUPPORTED),
    ({"scale": 0.0}, _hip.EINVAL),
    ({"scale": float("nan")}, _hip.EINVAL),
    ({"scale": float("inf")}, _hip.EINVAL),
    ({"bt_width": 6}, _hip.EINVAL),  # 96 tokens
    ({"masks": None}, _hip.EINVAL),
    ({"num_blocks": 0}, _hip.EINVAL),
    ({"q": PTR + 8}, _hip.EINVAL),
    ({"q_stride_h": 68}, _hip.EINVAL),
    ({"out": PTR + 2}, _hip.EINVAL),
    ({"k_cache": PTR + 4}, _hip.EINVAL),
    ({"kv_stride_n": 1 << 31}, _hip.EUNSUPPORTED),
    ({"kv_mode": 1, "k_scale": None}, _hip.EINVAL),
    ({"kv_mode": 1, "k_scale_dtype": _hip.BF16}, _hip.EUNSUPPORTED),
    ({"kv_mode": 1, "v_scale": PTR + 1}, _hip.EINVAL),
    ({"max_context": 4096, "bt_width": 256, "num_splits": 4, "workspace": None}, _hip.EWORKSPACE),
    ({"max_context": 4096, "bt_width": 256, "num_splits": 4, "workspace": PTR + 128, "workspace_bytes": 1 << 30}, _hip.EWORKSPACE),
])
def test_tree_attention_refuses(over, code):
    assert _hip.lib().sipa_tree_attention(ctypes.byref(tree(**over)), None) == code, _hip.lib().sipa_last_error()


def test_tree_attention_of_nothing():
    lib = _hip.lib()
    assert lib.sipa_tree_attention(ctypes.byref(tree(num_seqs=0)), None) == 0
    assert lib.sipa_tree_attention(ctypes.byref(tree(num_tokens=0)), None) == 0


@pytest.mark.parametrize("head_dim,nodes,most", [(64, 4, 128), (64, 256, 40), (128, 4, 128), (128, 256, 72)])
def test_contexts_past_the_merges_splits_are_refused(head_dim, nodes, most):
    # A split holds 16384 keys at most and the merge keeps m and l of every split of a row group in the tile buffers: 2
    # stages x K and V x keys of a stage x (head_dim + 16) x 2 bytes, 8 bytes a row and split, 128 splits at most.
    def bytes_of(context, splits):
        p = tree(head_dim=head_dim, max_nodes=nodes, words=4, max_context=context, num_splits=splits, num_seqs=1)
        counters = ctypes.c_int64()
        return _hip.lib().sipa_tree_workspace_bytes(ctypes.byref(p), ctypes.byref(counters)), counters.value

    for splits in (1, most, 1000):
        total, counters = bytes_of(most * 16384, splits)
        assert total > counters > 0
        assert bytes_of(most * 16384 + 1, splits)[0] == _hip.EUNSUPPORTED
    assert bytes_of(100, 1) == (0, 0)


def maps(**over):
    base = dict(num_seqs=2, num_tokens=8, block_size=16, out_width=4, words=1, table_rows=4, table_width=8, table_stride=8)
    return filled(_hip.TreeMapsParams, **{**base, **over})


@pytest.mark.parametrize("over", [
    {"struct_size": 8}, {"num_seqs": 0}, {"num_seqs": 8193}, {"num_tokens": 0}, {"words": 0}, {"words": 5}, {"block_size": 0},
    {"out_width": 0}, {"table_rows": 0}, {"table_width": 0}, {"table_stride": 7}, {"parents": None}, {"ancestors": None},
])
def test_tree_maps_refuse(over):
    assert _hip.lib().sipa_tree_maps(ctypes.byref(maps(**over)), None) == _hip.EINVAL


def commit(**over):
    base = dict(num_layers=2, num_kv_heads=2, num_blocks=64, block_size=16, row_bytes=128, num_seqs=2, max_accepted=3, bt_width=4,
                k_stride_l=1 << 20, k_stride_h=1 << 17, v_stride_l=1 << 20, v_stride_h=1 << 17, bt_stride_s=4, acc_stride_s=3)
    return filled(_hip.CommitParams, **{**base, **over})


@pytest.mark.parametrize("over,code", [
    ({"struct_size": 8}, _hip.EINVAL),
    ({"num_layers": 0}, _hip.EINVAL),
    ({"max_accepted": -1}, _hip.EINVAL),
    ({"bt_width": 0}, _hip.EINVAL),
    ({"row_bytes": 24}, _hip.EUNSUPPORTED),
    ({"row_bytes": 0}, _hip.EUNSUPPORTED),
    ({"accepted": None}, _hip.EINVAL),
    ({"v_scale": None}, _hip.EINVAL),
    ({"k_pool": PTR + 8}, _hip.EINVAL),
    ({"v_stride_h": 8}, _hip.EINVAL),
])
def test_commit_refuses(over, code):
    assert _hip.lib().sipa_commit_tokens(ctypes.byref(commit(**over)), None) == code


def test_commit_of_nothing():
    assert _hip.lib().sipa_commit_tokens(ctypes.byref(commit(num_seqs=0)), None) == 0
    assert _hip.lib().sipa_commit_tokens(ctypes.byref(commit(max_accepted=0)), None) == 0


def logits(**over):
    base = dict(num_rows=2, vocab=1000, num_seqs=2, dtype=_hip.BF16, words=1, logits_stride=1000, out_stride=1000, history_size=10,
                num_biases=4, grammar_stride=32, grammar_states=2)
    return filled(_hip.LogitsParams, **{**base, **over})


@pytest.mark.parametrize("over,code", [
    ({"struct_size": 8}, _hip.EINVAL),
    ({"num_rows": -1}, _hip.EINVAL),
    ({"num_seqs": 0}, _hip.EINVAL),
    ({"vocab": 0}, _hip.EINVAL),
    ({"vocab": (1 << 25) + 1}, _hip.EINVAL),  # tiles of 1024 fp32 logits, at most 65535 of them in a grid's second dimension
    ({"dtype": 99}, _hip.EUNSUPPORTED),
    ({"logits": None}, _hip.EINVAL),
    ({"history_starts": None}, _hip.EINVAL),
    ({"masks": None}, _hip.EINVAL),
    ({"words": 0}, _hip.EINVAL),
    ({"words": 5}, _hip.EINVAL),
    ({"bias_values": None}, _hip.EINVAL),
    ({"history_size": -1}, _hip.EINVAL),
    ({"num_biases": -1}, _hip.EINVAL),
    ({"grammar": None}, _hip.EINVAL),
    ({"grammar_states": 0}, _hip.EINVAL),
    ({"grammar_stride": 31}, _hip.EINVAL),
])
def test_logits_refuse(over, code):
    assert _hip.lib().sipa_adjust_logits(ctypes.byref(logits(**over)), None) == code


def test_logits_of_nothing():
    assert _hip.lib().sipa_adjust_logits(ctypes.byref(logits(num_rows=0)), None) == 0


def test_no_capture_on_the_default_stream():
    assert _hip.lib().sipa_capture_id(None) == 0
