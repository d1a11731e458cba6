"""Selections of more rows or requests than a launch holds threads for are refused by their sizes. CPU."""

import ctypes

import pytest

from engine import _hip

GOOD = dict(num_rows=8, vocab=100, num_groups=2, beams=4, num_candidates=1, dtype=_hip.BF16)


def workspace(**over):
    p = _hip.BeamParams(struct_size=ctypes.sizeof(_hip.BeamParams), **{**GOOD, **over})
    return _hip.lib().sipa_beam_workspace_bytes(ctypes.byref(p))


@pytest.mark.parametrize("over", [dict(num_rows=(1 << 24) - 1), dict(num_rows=(1 << 20) - 1, vocab=16 * 16384), dict(num_groups=(1 << 23) - 1),
                                  dict(num_rows=(1 << 20) - 1, vocab=16 * 8192, dtype=_hip.F32)])
def test_sizes_that_fit(over):
    assert workspace(**over) > 0


@pytest.mark.parametrize("over", [dict(num_rows=1 << 24), dict(num_rows=1 << 20, vocab=16 * 16384), dict(num_groups=1 << 23),
                                  dict(num_rows=1 << 20, vocab=16 * 8192, dtype=_hip.F32), dict(num_rows=(1 << 31) - 1),
                                  dict(num_groups=(1 << 31) - 1)])
def test_sizes_past_a_launch(over):
    assert workspace(**over) == _hip.EUNSUPPORTED
    # the call itself refuses before it looks for a workspace
    p = _hip.BeamParams(struct_size=ctypes.sizeof(_hip.BeamParams),
                        **{**GOOD, **over, **dict.fromkeys(("logits", "scores", "out_scores", "out_beams", "out_tokens", "starts"), 4096)})
    assert _hip.lib().sipa_beam_select(ctypes.byref(p), None) == _hip.EUNSUPPORTED
