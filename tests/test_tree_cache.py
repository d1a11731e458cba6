"""Drafted trees through the caches and the model: metadata from the host and from the device, the forward over trees, rules
on its logits, the commit of an accepted path and the decode that follows, as a speculative serving step uses them together.
On the CPU in fp32 (gather backend) and on the GPU (HIP kernels).

Tolerances: fp32 on the CPU, two forwards of the same tokens in other shapes: sums of at most 512 products in another order
through two layers, 1e-4 of the largest logit. bf16 on the GPU: two layers round to bf16 at about 12 places (norms,
projections, attention, activations, residuals), each by 1.6e-3 of the value in root mean square (a uniform error of up to half
a step, 2^-9 to 2^-8 of it); where the two forwards' sums differ in a last bit the roundings are independent, so the hidden
states differ by up to sqrt(2 * 12) * 1.6e-3 = 7.9e-3 and with them the logits, of their own root mean square, which is the
largest of some 10^3 to 10^4 logits over 3.5: 2.3e-3 of the largest logit, 1.8e-3 in the mean (0.8 of it), and the logits' own
two roundings add 5e-4. Allowed: 4e-3 in the mean, twice that, and 0.02 at most (4.5 times the root mean square is 0.010, the
largest logit's rounding 2^-8). The gather backend, which also takes the prompts of pools with other than 16-token blocks,
rounds scores to bf16 as well: 0.05 and 5e-3. INT8 caches quantize K and V of the two forwards apart: values that differ by
7.9e-3 of their root mean square, which is 1 / 2.7 of a row's largest, so by 0.37 of a code's step (1 / 127 of the largest),
get another code with that probability, a step off each: 0.6 steps or 1.3e-2 of the root mean square more, 1.5e-2 together.
That is the error of the attention's V and, once more, of its K: 2.1e-2 of the attention's output, and 2.3e-2 of the logits'
root mean square with the roundings above, 5.2e-3 of the largest logit in the mean. Allowed: twice that, 1e-2, and 0.05 at
most."""

import numpy as np
import pytest
import torch

from cases import fragmented_manager
from engine.block_manager import BlockManager
from engine.config import ModelConfig
from engine.device_tables import DeviceBlockTables
from engine.hip_logits import LogitsRules
from engine.model import Qwen2Model
from engine.paged_cache import PagedKVCache, TreeMetadata, build_metadata, build_tree_metadata
from engine.quant_cache import QuantPagedKVCache
from tree_cases import ancestor_sets, mask_tensor, random_parents

SMALL = ModelConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_layers=2, num_q_heads=4, num_kv_heads=2,
                    head_dim=16)
GPU = ModelConfig(vocab_size=512, hidden_size=896, intermediate_size=512, num_layers=2, num_q_heads=14, num_kv_heads=2,
                  head_dim=64)


def close(a, b, frac, mean_frac, what):
    a, b = a.float(), b.float()
    scale = b.abs().max().item()
    err = (a - b).abs()
    assert err.max().item() <= frac * scale, f"{what}: max {err.max().item():.3e} of scale {scale:.3e}"
    assert err.mean().item() <= mean_frac * scale, f"{what}: mean {err.mean().item():.3e} of scale {scale:.3e}"


def new_cache(cfg, m, device, fmt="bf16", backend=None):
    backend = backend or ("gather" if device == "cpu" else "hip")
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    if fmt == "bf16":
        return PagedKVCache(cfg, m.num_blocks, m.block_size, device, dtype, backend)
    return QuantPagedKVCache(cfg, m.num_blocks, m.block_size, device, dtype, backend, fmt, m, n_stage=16)


def setup(device, fmt="bf16", backend=None, block=16, seed=0):
    cfg = SMALL if device == "cpu" else GPU
    m = fragmented_manager(200, block, torch.Generator().manual_seed(seed))
    model = Qwen2Model(cfg, device, torch.float32 if device == "cpu" else torch.bfloat16, seed=1, max_positions=1024, std=0.1)
    return cfg, m, model, new_cache(cfg, m, device, fmt, backend)


def prefill(model, cache, m, prompts, device):
    for s, p in enumerate(prompts):
        m.allocate(s, len(p))
    meta = build_metadata(m, [(s, 0, len(p)) for s, p in enumerate(prompts)], device)
    return model.forward(torch.cat(prompts), meta.positions, cache, meta)


def path_logits(cfg, model, device, fmt, prompt, path, backend=None):
    """Logits after the last token of prompt + path, from the prompt and one chunk on a cache of their own."""
    m = BlockManager(64, 16)
    cache = new_cache(cfg, m, device, fmt, backend)
    prefill(model, cache, m, [prompt], device)
    m.append_slots(0, len(path))
    meta = build_metadata(m, [(0, len(prompt), len(path))], device)
    return model.forward(path, meta.positions, cache, meta)[0]


CASES = [("cpu", "bf16", None, 16), ("cpu", "int8", None, 16)] + [
    pytest.param("cuda", f, b, n, marks=pytest.mark.gpu)
    for f, b, n in (("bf16", "hip", 16), ("bf16", "triton", 32), ("bf16", "gather", 16), ("int8", "hip", 16),
                    ("int8", "hip", 64))]


def tolerance(device, fmt, backend, block):
    if device == "cpu":
        return (1e-4, 1e-4) if fmt == "bf16" else (0.05, 5e-3)
    if fmt == "int8":
        return 0.05, 1e-2
    return (0.02, 4e-3) if backend != "gather" and block == 16 else (0.05, 5e-3)


@pytest.mark.parametrize("device,fmt,backend,block", CASES)
def test_forward_commit_and_decode(device, fmt, backend, block):
    """Every node's logits are those of its path alone; after the commit of a path the sequence goes on as if the path had
    been decoded token by token."""
    cfg, m, model, cache = setup(device, fmt, backend, block)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).to(device) for n in (37, 16, 100)]
    prefill(model, cache, m, prompts, device)
    rng = np.random.RandomState(4)
    parents = [random_parents(n, rng) for n in (9, 1, 20)]
    parents[0] = [-1, 0, 0, 1, 2, 4, -1, 5, 7]
    ids = [torch.randint(0, cfg.vocab_size, (len(p),), generator=g).to(device) for p in parents]
    for s, p in enumerate(parents):
        m.append_slots(s, len(p))
    meta = build_tree_metadata(m, [(s, len(prompts[s]), parents[s]) for s in range(3)], device)
    logits = model.forward(torch.cat(ids), meta.positions, cache, meta)
    assert logits.shape == (30, cfg.vocab_size)
    frac, mean = tolerance(device, fmt, backend, block)
    want = []
    for s, p in enumerate(parents):
        for nodes in ancestor_sets(p):
            want.append(path_logits(cfg, model, device, fmt, prompts[s], ids[s][sorted(nodes)], backend))
    close(logits, torch.stack(want), frac, mean, "nodes")
    # the accepted paths: a branch whose nodes move, nothing, and the deepest node's
    deepest = max(ancestor_sets(parents[2]), key=len)
    accepted = [[0, 2, 4, 5, 7], [], sorted(deepest)]
    cache.commit(accepted)
    for s, a in enumerate(accepted):
        m.truncate(s, len(prompts[s]) + len(a))
    m.check_invariants()
    for s in range(3):
        m.append_slot(s)
    nxt = torch.randint(0, cfg.vocab_size, (3,), generator=g).to(device)
    meta = build_metadata(m, [(s, m.seq_len(s) - 1, 1) for s in range(3)], device)
    got = model.forward(nxt, meta.positions, cache, meta)
    want = [path_logits(cfg, model, device, fmt, prompts[s], torch.cat([ids[s][accepted[s]], nxt[s:s + 1]]), backend)
            for s in range(3)]
    close(got, torch.stack(want), frac, mean, "after the commit")


@pytest.mark.parametrize("device,fmt,backend,block", CASES)
def test_commit_moves_the_pools_rows(device, fmt, backend, block):
    cfg, m, model, cache = setup(device, fmt, backend, block)
    for s, n in enumerate((20, 7)):
        m.allocate(s, n + 12)
    pools = [t for t in (cache.k, cache.v, getattr(cache, "k_scale", None), getattr(cache, "v_scale", None)) if t is not None]
    g = torch.Generator().manual_seed(5)
    for t in pools:
        t.copy_(torch.randint(-100, 100, t.shape, generator=g))
    before = [t.clone() for t in pools]
    meta = build_tree_metadata(m, [(0, 20, [-1] * 12), (1, 7, list(range(-1, 11)))], device)
    cache.begin(meta.num_tokens, meta)
    accepted = [[1, 2, 3, 9], [0, 1, 5, 6, 7, 8, 11]]
    cache.commit(accepted)
    for t, b in zip(pools, before):
        for s, (start, path) in enumerate(zip((20, 7), accepted)):
            at = m.slots(s, 0, m.seq_len(s))
            for j, node in enumerate(path):
                to, frm = at[start + j], at[start + node]
                b[:, :, to // block, to % block] = b[:, :, frm // block, frm % block]
        assert torch.equal(t, b)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rules_count_each_nodes_path(device):
    """The rules of a forward over trees: a node's logits are those of its path with the path's tokens as generated ones."""
    cfg, m, model, cache = setup(device)
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).to(device) for n in (12, 30)]
    prefill(model, cache, m, prompts, device)
    parents = [[-1, 0, 1, 0], [-1, 0, 0, 2, 3]]
    ids = [torch.randint(0, cfg.vocab_size, (len(p),), generator=g).to(device) for p in parents]
    ids[1][3] = ids[1][0]  # a token twice on a path
    for s, p in enumerate(parents):
        m.append_slots(s, len(p))
    f = lambda x: torch.tensor(x, device=device)  # noqa: E731
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    rules = LogitsRules(cfg.vocab_size, 2, history=torch.cat(prompts).int(), history_starts=f([0, 12, 42]),
                        prompt_lens=i([12, 25]), repetition=f([1.5, 1.2]), frequency=f([0.25, 0.5]), presence=f([0.5, 0.0]))
    batch = [(s, len(prompts[s]), parents[s]) for s in range(2)]
    meta = build_tree_metadata(m, batch, device)
    grammar = torch.randint(-(1 << 31), 1 << 31, (2, -(-cfg.vocab_size // 32)), generator=g).int().to(device)
    rules_g = LogitsRules(cfg.vocab_size, 2, grammar=grammar)
    raw = model.forward(torch.cat(ids), meta.positions, cache, meta)
    got = model.forward(torch.cat(ids), meta.positions, cache, meta, rules=rules)
    states = i([0, 1, -1, 0, 1, 0, -1, 1, 1])
    masked = model.forward(torch.cat(ids), meta.positions, cache, meta, rules=rules_g, grammar_rows=states)
    row = 0
    for s, p in enumerate(parents):
        for nodes in ancestor_sets(p):
            history = torch.cat([prompts[s], ids[s][sorted(nodes)]]).int()
            alone = LogitsRules(cfg.vocab_size, 1, history=history, history_starts=f([0, len(history)]),
                                prompt_lens=rules.prompt_lens[s:s + 1], repetition=rules.repetition[s:s + 1],
                                frequency=rules.frequency[s:s + 1], presence=rules.presence[s:s + 1])
            assert torch.equal(got[row], alone.apply(raw[row:row + 1])[0])
            st = int(states[row])
            v = torch.arange(cfg.vocab_size, device=device)
            ok = torch.ones_like(v, dtype=torch.bool) if st < 0 else (grammar[st][v // 32] >> (v % 32) & 1).bool()
            assert torch.equal(masked[row], raw[row].masked_fill(~ok, float("-inf")))
            row += 1


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rules_of_ordinary_forwards(device):
    cfg, m, model, cache = setup(device)
    prompts = [torch.arange(5, 5 + n, device=device) for n in (9, 4)]
    for s, p in enumerate(prompts):
        m.allocate(s, len(p))
    meta = build_metadata(m, [(0, 0, 9), (1, 0, 4)], device)
    rules = LogitsRules(cfg.vocab_size, 2, history=torch.cat(prompts).int(),
                        history_starts=torch.tensor([0, 9, 13], device=device),
                        repetition=torch.tensor([2.0, 3.0], device=device))
    ids = torch.cat(prompts)
    raw = model.forward(ids, meta.positions, cache, meta)
    assert torch.equal(model.forward(ids, meta.positions, cache, meta, rules=rules), rules.apply(raw))
    every = model.forward(ids, meta.positions, cache, meta, last_only=False)
    starts = torch.tensor([0, 9, 13], dtype=torch.int32, device=device)
    assert torch.equal(model.forward(ids, meta.positions, cache, meta, last_only=False, rules=rules),
                       rules.apply(every, query_starts=starts))


def test_tree_metadata_matches_the_definition():
    m = fragmented_manager(300, 16, torch.Generator().manual_seed(7))
    rng = np.random.RandomState(8)
    batch = []
    for s, (start, n) in enumerate([(0, 1), (15, 3), (100, 65), (33, 256), (5, 128)]):
        m.allocate(s, start + n + s)
        batch.append((s, start, random_parents(n, rng)))
    meta = build_tree_metadata(m, batch, "cpu")
    base = build_metadata(m, [(s, a, len(p)) for s, a, p in batch], "cpu")
    sets = [x for _, _, p in batch for x in ancestor_sets(p)]
    starts = [a for _, a, p in batch for _ in p]
    assert isinstance(meta, TreeMetadata) and meta.max_nodes == 256 and meta.starts() == [a for _, a, _ in batch]
    assert torch.equal(meta.masks, mask_tensor(sets, 4))
    assert meta.positions.tolist() == [a + len(x) - 1 for a, x in zip(starts, sets)]
    assert meta.query_starts_t.tolist() == meta.query_starts == base.query_starts
    for f in ("slot_mapping", "slot_blocks", "slot_offsets", "block_tables", "context_lens_t", "last_token_indices"):
        assert torch.equal(getattr(meta, f), getattr(base, f)), f


@pytest.mark.gpu
def test_device_tables_derive_the_same_metadata():
    m = fragmented_manager(3000, 16, torch.Generator().manual_seed(9))
    dt = DeviceBlockTables(m, "cuda", max_seqs=40, max_blocks=64)
    rng = np.random.RandomState(10)
    for s in range(30):
        m.allocate(s, int(rng.randint(1, 600)))
    for step in range(6):
        batch = []
        for s in rng.permutation(30)[:rng.randint(1, 31)].tolist():
            n = int(rng.randint(1, 70))
            batch.append((s, m.seq_len(s), random_parents(n, rng)))
            m.append_slots(s, n)
        dev, host = dt.build_tree(batch), build_tree_metadata(m, batch, "cuda")
        for f in ("positions", "slot_mapping", "slot_blocks", "slot_offsets", "block_tables", "context_lens_t",
                  "last_token_indices", "masks", "query_starts_t"):
            a, b = getattr(dev, f), getattr(host, f)
            assert a.dtype == b.dtype and torch.equal(a, b), f
        assert dev.query_starts == host.query_starts and dev.context_lens == host.context_lens
        assert dev.parents == host.parents and list(dev.slots_cpu) == list(host.slots_cpu)
        assert [x for x in dev.block_ids_cpu] == [x for x in host.block_ids_cpu]
        for s, start, p in batch:  # part of each tree is accepted, the rest given up
            m.truncate(s, min(start + int(rng.randint(0, len(p) + 1)), 600))
        m.check_invariants()
    with pytest.raises(ValueError):
        dt.build_tree([])
    with pytest.raises(ValueError):
        dt.build_tree([(0, m.seq_len(0), [-1])])
    with pytest.raises(ValueError):
        dt.build_tree([(0, 0, [0])])


@pytest.mark.gpu
def test_graph_runner_steps_with_rules():
    from engine.graph_runner import DecodeGraphRunner

    cfg, m, model, cache = setup("cuda")
    prompts = [torch.arange(3, 3 + n, device="cuda") for n in (20, 33, 5)]
    prefill(model, cache, m, prompts, "cuda")
    runner = DecodeGraphRunner(model, cache, m, max_batch=4, max_context=64)
    rules = LogitsRules(cfg.vocab_size, 3, history=torch.cat(prompts).int(),
                        history_starts=torch.tensor([0, 20, 53, 58], device="cuda"),
                        frequency=torch.tensor([1.0, 2.0, 3.0], device="cuda"))
    for step in range(3):
        for s in range(3):
            m.append_slot(s)
        ids = torch.tensor([7, 8, 9 + step], device="cuda")
        raw = runner.step([0, 1, 2], ids).clone()
        got = runner.step([0, 1, 2], ids, rules=rules)
        assert torch.equal(got, rules.apply(raw)) and not torch.equal(got, raw)
        assert torch.equal(runner.step([0, 1, 2], ids), raw)  # the graph's own logits are left alone
    runner.close()


def test_truncate():
    m = fragmented_manager(20, 16, torch.Generator().manual_seed(11))
    freed = []
    m.add_free_listener(lambda blocks: freed.append(list(blocks)))
    m.allocate(0, 100)
    table = m.block_table(0)
    free = m.num_free_blocks()
    m.truncate(0, 50)
    assert m.block_table(0) == table[:4] and m.seq_len(0) == 50 and m.num_free_blocks() == free + 3
    assert freed[-1] == table[4:][::-1]
    m.check_invariants()
    m.append_slots(0, 40)  # the blocks come back in table order
    assert m.block_table(0) == table[:6]
    m.truncate(0, 90), m.truncate(0, 0)
    assert m.block_table(0) == [] and m.seq_len(0) == 0
    m.check_invariants()
    for n in (-1, 1):
        with pytest.raises(ValueError):
            m.truncate(0, n)


def test_refusals():
    m = BlockManager(64, 16)
    m.allocate(0, 40)
    build_tree_metadata(m, [(0, 30, [-1] * 10)], "cpu")
    for batch in ([(0, 30, [])], [(0, 30, [0])], [(0, 30, [-1, 1])], [(0, 30, [-1, -2])], [(0, 30, [-1] * 11)],
                  [(0, -1, [-1])], [], [(0, 0, [-1] * 257)]):
        with pytest.raises(ValueError):
            build_tree_metadata(m, batch, "cpu")
    cache = new_cache(SMALL, m, "cpu")
    meta = build_tree_metadata(m, [(0, 30, [-1, 0, 0])], "cpu")
    cache.begin(3, meta)
    for accepted in ([[1, 0]], [[0, 0]], [[3]], [[-1]], [[0], [0]], []):
        with pytest.raises(ValueError):
            cache.commit(accepted)
    cache.commit([[]])
    cache.begin(10, build_metadata(m, [(0, 30, 10)], "cpu"))
    with pytest.raises(ValueError):
        cache.commit([[0]])
    kchan = QuantPagedKVCache(SMALL, 64, 16, "cpu", torch.float32, "gather", "int8-kchannel", m, n_stage=4)
    with pytest.raises(ValueError):
        kchan.begin(3, meta)
    hip = PagedKVCache(SMALL, 64, 16, "cpu", torch.float32, "hip")
    with pytest.raises(ValueError):
        hip.begin(3, meta)
