"""Tree attention (engine/hip_tree.py TreePlan, sipa_tree_attention) against the definition in 64 bits: trees of one node to
the limit, contexts from none to several splits, odd groups, block sizes, both pool formats, strided rows, masks that leave
rows empty, garbage in hidden places, graphs and streams."""

import pytest
import torch

from engine.hip_tree import TreePlan, paged_tree_attention
from tree_cases import Case

pytestmark = pytest.mark.gpu


def attend(c: Case, **kw):
    return paged_tree_attention(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes,
                                quant=c.quant(), **kw)


def check(c: Case, got: torch.Tensor, ref=None):
    out, tol = ref or c.reference()
    err = (got.cpu().double() - out).abs()
    worst = (err - tol).max().item() if err.numel() else 0
    assert not torch.isnan(got).any() and worst <= 0, f"error past the bound by {worst}, largest error {err.max().item()}"


HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "mha": (3, 3, 64), "wide": (34, 2, 128), "one": (64, 1, 64)}
BATCHES = {
    "one_node": [(0, 1), (1, 1), (15, 1), (16, 1), (200, 1)],
    "small": [(5, 4), (31, 2), (0, 3), (100, 7)],
    "odd": [(333, 13), (64, 9), (1, 33)],
    "words": [(40, 64), (17, 65)],
}


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("batch", BATCHES)
def test_attention_matches_the_definition(batch, heads, int8):
    c = Case(BATCHES[batch], HEADS[heads], int8=int8, seed=len(batch) + len(heads))
    print(batch, heads, int8, flush=True)
    check(c, attend(c))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("splits", [None, 1, 2, 7])
def test_blocks_and_splits(block, splits, int8):
    c = Case([(700, 5), (3, 11), (513, 1), (0, 20)], HEADS["1.5b" if block == 32 else "0.5b"], block, int8, seed=block)
    print(block, splits, int8, flush=True)
    check(c, attend(c, num_splits=splits))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("splits", [None, 2, 3, 7, 13])
@pytest.mark.parametrize("seqs,heads", [(1, (7, 1, 64)), (1, (14, 2, 64)), (3, (6, 1, 128)), (2, (4, 2, 128)), (5, (6, 2, 64)),
                                        (9, (2, 1, 64)), (9, (14, 2, 64))])
def test_splits_on_one_or_several_xcds(seqs, heads, splits, int8):
    # 1, 2, 3 and 4, up to 16 and more pairs of a sequence and a KV head; row groups where the trees are large. The merge
    # reads splits in their order: a second call on the plan's workspace gives the same bits.
    c = Case([(1500 - 97 * i, 5 + 9 * (i % 3)) for i in range(seqs)], heads, int8=int8, seed=seqs)
    print(seqs, heads, splits, int8, flush=True)
    plan = TreePlan(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes, quant=c.quant(),
                    num_splits=splits)
    first = plan(c.q, c.k, c.v)
    check(c, first)
    for _ in range(3):
        assert torch.equal(plan(c.q, c.k, c.v), first)


def test_largest_trees():
    c = Case([(50, 256), (0, 255), (1000, 129)], (2, 2, 64), seed=3)
    check(c, attend(c))
    check(c, attend(c, num_splits=4))


@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.float32])
def test_int8_scale_types(scale_dtype):
    c = Case([(90, 6), (300, 3)], HEADS["0.5b"], int8=True, seed=5, scale_dtype=scale_dtype)
    check(c, attend(c, num_splits=2))


@pytest.mark.parametrize("int8", [False, True])
def test_rows_that_see_nothing_are_zero(int8):
    # no cached token, and masks that are empty, of the row alone, or of a later node alone
    seqs = [(0, 4), (0, 3), (6, 2)]
    sets = [set(), {1}, {3}, {0, 2}, set(), set(), set(), {1}, {0}]
    c = Case(seqs, HEADS["0.5b"], int8=int8, seed=6, sets=sets)
    for splits in (None, 1):
        got = attend(c, num_splits=splits)
        check(c, got)
        for r in (0, 4, 5, 6):
            assert (got[r] == 0).all()


def test_long_context_with_empty_tree_masks_in_split_runs():
    sets = [set() for _ in range(5)]
    c = Case([(1500, 5)], HEADS["1.5b"], seed=7, sets=sets)
    check(c, attend(c, num_splits=5))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("splits", [1, 3])
def test_garbage_in_hidden_places(int8, splits):
    """Infinities and NaN in K, V and scales of nodes that a row does not see, past the context and in spare blocks."""
    c = Case([(37, 9), (0, 6), (200, 5)], HEADS["0.5b"], int8=int8, seed=8)
    ref = c.reference()
    used = {int(b) for row in c.bt.cpu().tolist() for b in row if b >= 0}
    bad = float("nan")
    for i, (cached, n) in enumerate(c.seqs):
        last = int(c.bt[i, (cached + n - 1) // c.B])
        tail = slice((cached + n - 1) % c.B + 1, c.B)
        for t in ((c.ks, c.vs) if int8 else (c.k, c.v)):
            t[:, last, tail] = bad
    for b in set(range(c.N)) - used:
        for t in ((c.ks, c.vs) if int8 else (c.k, c.v)):
            t[:, b] = float("inf")
    # a node that only itself sees holds garbage: every other row keeps its result
    at, spoiled = 0, []
    for i, (cached, n) in enumerate(c.seqs):
        leaf = n - 1
        if all(leaf not in c.sets[at + r] for r in range(n - 1)):
            p = cached + leaf
            blk, off = int(c.bt[i, p // c.B]), p % c.B
            for t, x in zip((c.ks, c.vs) if int8 else (c.k, c.v), (bad, float("inf"))):
                t[:, blk, off] = x
            spoiled.append(at + leaf)
        at += n
    assert spoiled
    got = attend(c, num_splits=splits)
    keep = [r for r in range(at) if r not in spoiled]
    check(c, got[keep], (ref[0][keep], ref[1][keep]))
    for r in spoiled:
        assert torch.isnan(got[r]).all()


def test_infinite_values_that_are_seen():
    """A row that sees an infinite V has it in its sum; the others do not."""
    c = Case([(20, 4)], (2, 1, 64), seed=9, chain=True)
    ref = c.reference()
    p = 20 + 2
    c.v[:, int(c.bt[0, p // 16]), p % 16, 5] = float("inf")
    got = attend(c)
    check(c, got[:2], (ref[0][:2], ref[1][:2]))
    assert torch.isinf(got[2:, :, 5]).all()
    keep = [i for i in range(64) if i != 5]
    check(c, got[2:][..., keep], (ref[0][2:][..., keep], ref[1][2:][..., keep]))


def test_strided_rows_and_rows_behind_the_last_sequence():
    c = Case([(60, 5), (9, 3)], HEADS["0.5b"], seed=10)
    ref = c.reference()
    T = c.q.shape[0]
    wide = torch.zeros(T + 4, 18 * 64, dtype=torch.bfloat16, device="cuda")
    q = wide[:, :14 * 64].view(T + 4, 14, 64)
    q[:T] = c.q
    masks = torch.cat([c.masks, torch.full((4, c.words), -1, device="cuda")])
    buf = torch.full((T + 4, 16, 80), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, 1:15, 8:72]
    plan = TreePlan(q, c.k, c.v, c.bt, c.ctx, c.qs, masks, c.scale, c.max_ctx, c.max_nodes)
    got = plan(q, c.k, c.v, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(c, got[:T], ref)
    assert (buf[T:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 15] == 7).all()
    assert (buf[:, :, :8] == 7).all() and (buf[:, :, 72:] == 7).all()


def test_sequences_without_nodes():
    """Padding sequences of a captured batch: no rows, nothing read or written for them."""
    c = Case([(40, 3), (25, 0), (0, 2), (80, 0)], HEADS["0.5b"], seed=11)
    check(c, attend(c, num_splits=2))


def test_bad_ids_and_lengths_stay_inside():
    """Block ids outside the pool and lengths past max_context give wrong results, never an access outside (ids and lengths
    are clamped as in the decode kernels); the rows of the other sequence keep theirs."""
    c = Case([(100, 4), (50, 4)], HEADS["0.5b"], seed=12)
    ref = c.reference()
    c.bt[0, 2] = c.N + 1000
    c.bt[0, 3] = -7
    c.ctx[0] = 5000
    got = attend(c, num_splits=2)
    check(c, got[4:], (ref[0][4:], ref[1][4:]))


@pytest.mark.parametrize("int8", [False, True])
def test_far_blocks(int8):
    """Blocks past 2^32 elements of the pool."""
    heads = (2, 1, 128)
    c = Case([(100, 3)], heads, int8=int8, seed=13)
    ref = c.reference()
    per = 16 * 128
    N = (1 << 32) // per + 64
    far = N - c.N

    def move(t):
        big = torch.empty(1, N, *t.shape[2:], dtype=t.dtype, device="cuda")
        big[:, far:] = t
        return big

    c.k, c.v = move(c.k), move(c.v)
    if int8:
        c.ks, c.vs = move(c.ks), move(c.vs)
    c.bt = torch.where(c.bt >= 0, c.bt + far, c.bt)
    check(c, attend(c), ref)


def test_plan_runs_layers_and_new_tensors():
    c = Case([(70, 6), (20, 2)], HEADS["0.5b"], seed=14)
    d = Case([(70, 6), (20, 2)], HEADS["0.5b"], seed=15)
    plan = TreePlan(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes, num_splits=2)
    d.bt, d.masks, d.sets = c.bt, c.masks, c.sets
    check(d, plan(d.q, d.k, d.v))
    k, v = torch.stack([d.k, c.k]), torch.stack([d.v, c.v])
    check(c, plan.run_layer(1, c.q, k, v))
    check(d, plan.run_layer(-2, d.q, k, v))
    with pytest.raises(IndexError):
        plan.run_layer(2, c.q, k, v)


def test_graphs_and_streams_share_nothing():
    """One plan captured into two graphs and called eagerly on two streams at the same time: every result is its own."""
    c = Case([(900, 6), (500, 9), (40, 3)], HEADS["0.5b"], seed=16)
    ref = c.reference()
    plan = TreePlan(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes, num_splits=4)
    check(c, plan(c.q, c.k, c.v), ref)
    graphs = []
    for _ in range(2):
        out = torch.empty_like(c.q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):  # several layers of one forward
                plan(c.q, c.k, c.v, out=out)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for s, (g, out) in zip(streams, graphs):
            out.zero_()
        torch.cuda.synchronize()
        for s, (g, out) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(4):
                    g.replay()
        with torch.cuda.stream(streams[2]):
            outs.append(plan(c.q, c.k, c.v))
        torch.cuda.synchronize()
        for out in outs + [o for _, o in graphs]:
            check(c, out, ref)
        check(c, plan(c.q, c.k, c.v), ref)


def test_results_do_not_depend_on_the_run():
    c = Case([(3000, 16), (1200, 5)], HEADS["0.5b"], seed=17)
    plan = TreePlan(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes)
    first = plan(c.q, c.k, c.v)
    for _ in range(10):
        assert torch.equal(plan(c.q, c.k, c.v), first)


def test_a_chain_is_a_prefill_chunk_and_one_node_a_decode_row():
    """The same rows through the prefill and decode kernels, which meet the same bound."""
    from engine.hip_decode import paged_decode_attention
    from engine.hip_prefill import paged_prefill_attention

    c = Case([(300, 12), (77, 5)], HEADS["0.5b"], seed=18, chain=True)
    ref = c.reference()
    check(c, attend(c), ref)
    lens = c.qs[1:] - c.qs[:-1]
    pre = paged_prefill_attention(c.q, c.k, c.v, c.bt, c.ctx, c.qs[:-1].contiguous(), lens.contiguous(), c.scale, c.max_ctx,
                                  c.max_nodes)
    check(c, pre, ref)
    d = Case([(300, 1), (77, 1)], HEADS["0.5b"], seed=19)
    ref = d.reference()
    check(d, attend(d), ref)
    check(d, paged_decode_attention(d.q, d.k, d.v, d.bt, d.ctx, d.scale, d.max_ctx), ref)


def test_refusals():
    c = Case([(40, 3)], HEADS["0.5b"], seed=20)
    args = dict(q=c.q, k_cache=c.k, v_cache=c.v, block_tables=c.bt, context_lens=c.ctx, query_starts=c.qs, masks=c.masks,
                scale=c.scale, max_context=c.max_ctx, max_nodes=c.max_nodes)

    def refused(**over):
        with pytest.raises(ValueError):
            paged_tree_attention(**{**args, **over})

    refused(q=c.q.float())
    refused(q=c.q[:, :13])
    refused(q=c.q.transpose(1, 2))
    refused(k_cache=c.k.float(), v_cache=c.v.float())
    refused(k_cache=c.k[:, :, :8])
    refused(v_cache=c.v[:, :-1])
    refused(block_tables=c.bt.long())
    refused(max_context=c.max_ctx + 100)
    refused(context_lens=c.ctx.long())
    refused(query_starts=c.qs[:-1])
    refused(masks=c.masks.int())
    refused(masks=c.masks[:-1])
    refused(max_nodes=65)
    refused(max_nodes=0)
    refused(scale=0.0)
    refused(scale=float("nan"))
    refused(masks=c.masks.cpu())
    refused(out=torch.empty(3, 14, 64, device="cuda"))
    plan = TreePlan(*args.values())
    with pytest.raises(ValueError):
        plan(c.q[:2], c.k, c.v)
    with pytest.raises(ValueError):
        plan(c.q, c.k, c.v[:, :-1])
    i = Case([(40, 3)], HEADS["0.5b"], int8=True, seed=20)
    with pytest.raises(ValueError):
        paged_tree_attention(c.q, i.k, i.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, 3)
    from engine.hip_decode import QuantKV

    with pytest.raises(ValueError):
        paged_tree_attention(c.q, i.k, i.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, 3,
                             quant=QuantKV(2, i.ks, i.vs))
    with pytest.raises(ValueError):
        paged_tree_attention(c.q, i.k, i.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, 3,
                             quant=QuantKV(1, i.ks[:, :-1], i.vs))
