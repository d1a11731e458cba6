"""Rules given to a forward or to a step of the graph runner have to be those of its sequences: with others every row would
silently take another sequence's."""

import pytest
import torch

from engine.hip_logits import LogitsRules
from engine.paged_cache import build_metadata, build_tree_metadata
from test_tree_cache import prefill, setup

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def start(device):
    cfg, m, model, cache = setup(device)
    prefill(model, cache, m, [torch.arange(3, 3 + n, device=device) for n in (20, 9, 17)], device)
    rules = {n: LogitsRules(cfg.vocab_size, n, repetition=torch.full((n,), 2.0, device=device)) for n in (2, 3, 4)}
    return cfg, m, model, cache, rules


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["decode", "chunk", "every", "tree"])
def test_forwards_with_the_rules_of_other_sequences_are_refused(device, kind):
    cfg, m, model, cache, rules = start(device)
    n = 1 if kind == "decode" else 3
    lens = [m.seq_len(s) for s in range(3)]
    for s in range(3):
        m.append_slots(s, n)
    meta = build_tree_metadata(m, [(s, lens[s], [-1, 0, 0]) for s in range(3)], device) if kind == "tree" else \
        build_metadata(m, [(s, lens[s], n) for s in range(3)], device)
    ids = torch.arange(3 * n, device=device)
    before = cache.k.clone()
    for bad in (2, 4):
        with pytest.raises(ValueError, match="sequences"):
            model.forward(ids, meta.positions, cache, meta, last_only=kind != "every", rules=rules[bad])
    assert torch.equal(cache.k.view(torch.uint8), before.view(torch.uint8))  # refused before anything is written
    model.forward(ids, meta.positions, cache, meta, last_only=kind != "every", rules=rules[3])


@pytest.mark.gpu
def test_runner_steps_with_the_rules_of_other_sequences_are_refused():
    from engine.graph_runner import DecodeGraphRunner

    cfg, m, model, cache, rules = start("cuda")
    runner = DecodeGraphRunner(model, cache, m, max_batch=4, max_context=64)
    for s in range(3):
        m.append_slot(s)
    ids = torch.tensor([7, 8, 9], device="cuda")
    for bad in (2, 4):
        for graph in (True, False):
            with pytest.raises(ValueError, match="sequences"):
                runner.step([0, 1, 2], ids, graph=graph, rules=rules[bad])
    runner.step([0, 1, 2], ids, rules=rules[3])
    # a sequence leaves: the rules of three are no longer the batch's
    with pytest.raises(ValueError, match="sequences"):
        runner.step([0, 2], ids[:2], rules=rules[3])
    runner.step([0, 2], ids[:2], rules=rules[2])
    runner.close()


@pytest.mark.parametrize("device", DEVICES)
def test_paths_of_token_ids_in_any_integer_layout(device):
    """Token ids that the embedding takes, int32 or strided ones, are a tree's path too."""
    cfg, m, model, cache, rules = start(device)
    lens = [m.seq_len(s) for s in range(3)]
    for s in range(3):
        m.append_slots(s, 4)
    meta = build_tree_metadata(m, [(s, lens[s], [-1, 0, 1, 0]) for s in range(3)], device)
    ids = torch.arange(12, device=device) // 2
    want = model.forward(ids, meta.positions, cache, meta, rules=rules[3])
    assert not torch.equal(want, model.forward(ids, meta.positions, cache, meta))
    for other in (ids.int(), torch.stack([ids, ids], 1)[:, 0], torch.stack([ids.int(), ids.int()], 1)[:, 1]):
        assert torch.equal(model.forward(other, meta.positions, cache, meta, rules=rules[3]), want)


@pytest.mark.parametrize("device", DEVICES)
def test_grammar_states_without_rules_are_refused(device):
    """They would be ignored, and the logits come out unmasked."""
    cfg, m, model, cache, rules = start(device)
    lens = [m.seq_len(s) for s in range(3)]
    for s in range(3):
        m.append_slot(s)
    meta = build_metadata(m, [(s, lens[s], 1) for s in range(3)], device)
    states, ids = torch.zeros(3, dtype=torch.int32, device=device), torch.arange(3, device=device)
    with pytest.raises(ValueError, match="grammar"):
        model.forward(ids, meta.positions, cache, meta, grammar_rows=states)
    with pytest.raises(ValueError, match="grammar"):  # rules without a grammar
        model.forward(ids, meta.positions, cache, meta, rules=rules[3], grammar_rows=states)
    if device == "cuda":
        from engine.graph_runner import DecodeGraphRunner

        runner = DecodeGraphRunner(model, cache, m, max_batch=4, max_context=64)
        with pytest.raises(ValueError, match="grammar"):
            runner.step([0, 1, 2], ids, grammar_rows=states)
        runner.close()
