"""Beams that share blocks through the caches, the model and the graph runner on the GPU: every layer's attention of a beam search
against 64 bits on the cache's own contents, which are those of sequences that share nothing."""

import dataclasses
import random

import pytest
import torch

from engine.block_manager import BlockManager
from engine.config import ModelConfig
from engine.device_tables import DeviceBlockTables
from engine.graph_runner import DecodeGraphRunner
from engine.hip_beam import beam_select
from engine.hip_decode import DecodePlan
from engine.hip_prefix import PrefixPlan
from engine.model import Qwen2Model
from engine.paged_cache import PagedKVCache, build_metadata
from engine.quant_cache import QuantPagedKVCache

pytestmark = pytest.mark.gpu
CFG = ModelConfig(vocab_size=1031, hidden_size=448, intermediate_size=256, num_layers=2, num_q_heads=7, num_kv_heads=1, head_dim=64)
FORMATS = ["bf16", "int8", "int8-kchannel"]


def make_cache(fmt, m, backend="hip"):
    """A cache that takes the shared-prefix kernel however little is shared."""
    if fmt == "bf16":
        cache = PagedKVCache(CFG, m.num_blocks, m.block_size, "cuda", torch.bfloat16, backend)
    else:
        cache = QuantPagedKVCache(CFG, m.num_blocks, m.block_size, "cuda", torch.bfloat16, backend, fmt=fmt, manager=m, n_stage=64)
    cache.prefix_min_bytes = 1
    return cache


def contents(cache, layer, i):
    """Sequence i's K and V in float64, as the kernels read them (gather() rounds INT8 to bf16)."""
    meta, B = cache.meta, cache.block_size
    n, ids = meta.context_lens[i], meta.block_ids[i]
    k, v = cache.k[layer][:, ids].double(), cache.v[layer][:, ids].double()
    fmt = getattr(cache, "fmt", "bf16")
    if fmt != "bf16":
        v = v * cache.v_scale[layer][:, ids].double()[..., None]
        k = k * cache.k_scale[layer][:, ids].double().unsqueeze(-1 if fmt == "int8" else 2)
        if fmt == "int8-kchannel" and n % B:
            k[:, -1] = cache.stage[layer][:, cache._stage_of[meta.block_ids_cpu[i][-1]]].double()
    return tuple(t.reshape(t.shape[0], -1, t.shape[-1])[:, :n] for t in (k, v))


class Checked:
    """A cache whose decode attention is compared with 64 bits. Bounds as in prefix_cases.expected; the decode kernel over
    per-channel scales takes fp16 products of q and scale, and fp16 probabilities times V's scale (2^-11 each)."""

    def __init__(self, cache):
        self.cache, self.checked = cache, 0

    def begin(self, n, meta):
        self.cache.begin(n, meta)

    def write(self, layer, k, v):
        self.cache.write(layer, k, v)

    def attend(self, layer, q, positions, scale):
        out = self.cache.attend(layer, q, positions, scale)
        m = self.cache.meta
        rough = 2 ** -10 if getattr(self.cache, "fmt", "") == "int8-kchannel" else 0.
        for i, c in enumerate(m.context_lens):
            a = m.query_starts[i]
            if m.query_starts[i + 1] - a > 1:
                continue
            k, v = contents(self.cache, layer, i)
            x = q[a].double()
            kt = k[0].T.contiguous()
            w = torch.softmax(x @ kt * scale, -1)
            want, size = w @ v[0], w @ v[0].abs()
            score = (2 * 64 * 2 ** -24 + rough) * scale * (x.abs() @ kt.abs()).amax(-1, keepdim=True)
            rel = 2 * (score + 2 ** -18 + 2 ** -22 + 2 ** -15 + rough) + 2 * (c / 16 + 64) * 2 ** -24
            assert ((out[a].view(7, 64).double() - want).abs() <= 2 ** -8 * want.abs() + rel * size * (1 + 2 ** -8)).all()
            self.checked += 1
        return out


@pytest.mark.parametrize("fmt", FORMATS)
def test_beam_search(fmt):
    """Two requests, four beams each, among a sequence that shares nothing: prompts prefilled once, beams forked, 40 steps."""
    K, steps = 4, 40
    model = Qwen2Model(CFG, "cuda", torch.bfloat16, seed=1, max_positions=512, std=0.05)
    m = BlockManager(200, 16)
    cache = make_cache(fmt, m)
    checked = Checked(cache)
    r = random.Random(2)
    prompts = {0: [r.randrange(1031) for _ in range(75)], 10: [r.randrange(1031) for _ in range(160)],
               99: [r.randrange(1031) for _ in range(30)]}
    for s, p in prompts.items():
        m.allocate(s, len(p))
    meta = build_metadata(m, [(s, 0, len(p)) for s, p in prompts.items()], "cuda")
    ids = torch.tensor([t for p in prompts.values() for t in p], device="cuda")
    logits = model.forward(ids, meta.positions, checked, meta)
    choice = beam_select(logits[:2], torch.zeros(2, device="cuda"), 1, K)
    seqs = [0, 1, 2, 3, 10, 11, 12, 13]
    copies = m.fork(0, [1, 2, 3])
    copies += m.fork(10, [11, 12, 13])
    assert len(copies) == 3  # the second prompt ends at a block's end
    cache.copy_blocks(copies)
    scores, tokens = choice.scores.reshape(-1), choice.tokens.reshape(-1)
    other, kinds, moved = logits[2].argmax(), set(), 0
    for _ in range(steps):
        batch = seqs + [99]
        for s in batch:
            m.append_slot(s)
        meta = build_metadata(m, [(s, m.seq_len(s) - 1, 1) for s in batch], "cuda")
        assert sorted(rows for rows, _ in meta.shared) == [[0, 1, 2, 3], [4, 5, 6, 7]] or moved
        logits = model.forward(torch.cat([tokens, other[None]]), meta.positions, checked, meta)
        kinds.add(type(cache._plan))
        choice = beam_select(logits[:8].contiguous(), scores, K, K)
        cpu = beam_select(logits[:8].cpu(), scores.cpu(), K, K)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(choice[1:], cpu[1:]))
        parents = (choice.beams + torch.arange(2, device="cuda")[:, None] * K).reshape(-1).tolist()
        moved += sum(p != i for i, p in enumerate(parents))
        cache.copy_blocks(m.reorder(seqs, parents))
        scores, tokens, other = choice.scores.reshape(-1), choice.tokens.reshape(-1), logits[8].argmax()
    m.check_invariants()
    assert moved > 10 and checked.checked == 2 * 9 * steps
    assert kinds == ({DecodePlan} if fmt == "int8-kchannel" else {PrefixPlan})
    for s in seqs + [99]:
        m.free(s)
    assert m.num_free_blocks() == 200 and not getattr(cache, "_stage_of", {})


@pytest.mark.parametrize("fmt", FORMATS)
def test_copied_blocks_hold_what_was_copied(fmt):
    m = BlockManager(40, 16)
    cache = make_cache(fmt, m)
    m.allocate(0, 37)
    meta = build_metadata(m, [(0, 0, 37)], "cuda")
    cache.begin(37, meta)
    k, v = (torch.randn(37, 1, 64, device="cuda").bfloat16() for _ in range(2))
    for layer in range(2):
        cache.write(layer, k, v)
    cache.copy_blocks(m.fork(0, [1, 2]))
    for s in (1, 2):
        m.append_slot(s)
        cache.begin(1, build_metadata(m, [(s, 37, 1)], "cuda"))
        for layer in range(2):
            cache.write(layer, k[s:s + 1], v[s:s + 1])
    got = []
    for s in (0, 1, 2):
        cache.meta = build_metadata(m, [(s, m.seq_len(s) - 1, 1)], "cuda") if s else meta
        got.append([contents(cache, layer, 0) for layer in range(2)])
    for s in (1, 2):
        for layer in range(2):
            for a, b in zip(got[0][layer], got[s][layer]):
                assert torch.equal(a, b[:, :37]) and not torch.equal(b[:, 37:], torch.zeros_like(b[:, 37:]))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_mixed_forwards(fmt):
    """Decode rows of groups among prefill chunks and rows of their own, in place and not: each as in a forward without
    groups, to what two kernels may differ by."""
    model = Qwen2Model(CFG, "cuda", torch.bfloat16, seed=1, max_positions=512, std=0.05)
    m = BlockManager(100, 16)
    cache = make_cache(fmt, m)
    for s, n in ((0, 100), (5, 64), (7, 20)):
        m.allocate(s, n)
        meta = build_metadata(m, [(s, 0, n)], "cuda")
        model.forward(torch.arange(n, device="cuda"), meta.positions, cache, meta)
    cache.copy_blocks(m.fork(0, [1, 2]) + m.fork(5, [6]))
    m.allocate(8, 33)
    for s in (0, 1, 2, 5, 6, 7):
        m.append_slot(s)
    decode = {s: (s, m.seq_len(s) - 1, 1) for s in (0, 1, 2, 5, 6, 7)}
    for order in ([0, 8, 1, 6, 7, 2, 5], [8, 0, 1, 2, 5, 6, 7], [0, 5, 1, 6, 2, 8]):
        batch = [decode[s] if s in decode else (8, 0, 33) for s in order]
        for build in (lambda: build_metadata(m, batch, "cuda"),
                      lambda: DeviceBlockTables(m, "cuda", 16, 16).build(batch)):
            meta = build()
            assert len(meta.shared) == 2
            g = torch.Generator(device="cuda").manual_seed(1)
            T = meta.num_tokens
            q = torch.randn(T, 7, 64, generator=g, device="cuda").bfloat16()
            k, v = (torch.randn(T, 1, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
            checked = Checked(cache)
            checked.begin(T, meta)
            checked.write(0, k, v), checked.write(1, k, v)
            for layer in range(2):
                out = checked.attend(layer, q, meta.positions, 0.125)
                assert type(cache._plan) is PrefixPlan and out.shape == (T, 448)
            assert checked.checked == 2 * (len(order) - (8 in order))


@pytest.mark.parametrize("fmt", FORMATS)
def test_graph_runner_over_beams(fmt):
    """Replayed steps over forked and reordered sequences: the device's block tables follow, and the logits are those of the
    static step run eagerly."""
    model = Qwen2Model(CFG, "cuda", torch.bfloat16, seed=1, max_positions=512, std=0.05)
    m = BlockManager(120, 16)
    cache = make_cache(fmt, m)
    m.allocate(0, 70)
    meta = build_metadata(m, [(0, 0, 70)], "cuda")
    logits = model.forward(torch.arange(70, device="cuda"), meta.positions, cache, meta)
    runner = DecodeGraphRunner(model, cache, m, 4, 256)
    seqs = [0, 1, 2, 3]
    choice = beam_select(logits, torch.zeros(1, device="cuda"), 1, 4)
    cache.copy_blocks(m.fork(0, seqs[1:]))
    with pytest.raises(ValueError, match="sequences hold"):
        m2 = BlockManager(8, 16)
        m2.allocate(0, 32)
        m2.fork(0, [1])
        m2.check_own(1, 31, 1)
    scores, tokens = choice.scores[0], choice.tokens[0]
    for step in range(20):
        for s in seqs:
            m.append_slot(s)
        got = runner.step(seqs, tokens).clone()
        for s in seqs:
            row = runner.tables.table[runner.tables.row(s)][:len(m.block_table(s))]
            assert row.tolist() == m.block_table(s)
        if fmt != "int8-kchannel":  # (a second step of the same token would stage it twice)
            assert torch.equal(got, runner.step(seqs, tokens, graph=False))
        choice = beam_select(got, scores, 4, 4)
        cache.copy_blocks(m.reorder(seqs, choice.beams[0].tolist()))
        scores, tokens = choice.scores[0], choice.tokens[0]
    runner.close()
    m.check_invariants()


def test_metadata_of_groups_is_kept_by_replace():
    m = BlockManager(20, 16)
    m.allocate(0, 32)
    m.fork(0, [1])
    for s in (0, 1):
        m.append_slot(s)
    meta = build_metadata(m, [(0, 32, 1), (1, 32, 1)], "cuda")
    assert meta.shared == [([0, 1], 32)]
    cache = make_cache("bf16", m)
    q = torch.randn(2, 7, 64, device="cuda").bfloat16()
    cache.k.normal_(), cache.v.normal_()
    outs = []
    for x in (meta, dataclasses.replace(meta, shared=[])):
        cache.begin(2, x)
        outs.append(cache.attend(0, q, x.positions, 0.125))
        outs.append(type(cache._plan))
    assert outs[1] is PrefixPlan and outs[3] is DecodePlan
    assert (outs[0].double() - outs[2].double()).abs().max() <= 2 ** -6 * outs[2].double().abs().max()


@pytest.mark.parametrize("fmt,rows,kernel", [("bf16", 384, DecodePlan), ("bf16", 386, PrefixPlan), ("int8", 743, DecodePlan),
                                             ("int8", 747, PrefixPlan)])
def test_the_kernel_is_chosen_by_what_is_shared(fmt, rows, kernel):
    """48 MiB that would be read again: 384 times 512 tokens of 256 bytes (bf16), 745 of 132 (INT8)."""
    m = BlockManager(32 + rows, 16)
    cache = make_cache(fmt, m)
    del cache.prefix_min_bytes
    m.allocate(0, 512)
    m.fork(0, list(range(1, rows)))
    for s in range(rows):
        m.append_slot(s)
    cache.k.zero_(), cache.v.zero_()
    meta = build_metadata(m, [(s, 512, 1) for s in range(rows)], "cuda")
    cache.begin(rows, meta)
    out = cache.attend(0, torch.zeros(rows, 7, 64, device="cuda").bfloat16(), meta.positions, 0.125)
    assert type(cache._plan) is kernel and out.shape == (rows, 448)


def test_metadata_without_groups():
    """An object with the reference's fields alone goes to the decode kernel."""
    m = BlockManager(20, 16)
    m.allocate(0, 33)
    meta = build_metadata(m, [(0, 32, 1)], "cuda")
    names = [f.name for f in dataclasses.fields(meta) if f.name != "shared"]
    bare = type("Bare", (), {**{n: getattr(meta, n) for n in names}, "num_seqs": 1})()
    cache = make_cache("bf16", m)
    cache.k.normal_(), cache.v.normal_()
    q = torch.randn(1, 7, 64, device="cuda").bfloat16()
    outs = []
    for x in (meta, bare):
        cache.begin(1, x)
        outs.append(cache.attend(0, q, x.positions, 0.125))
        assert type(cache._plan) is DecodePlan
    assert torch.equal(*outs)
