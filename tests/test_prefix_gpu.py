"""The shared-prefix attention kernel against 64 bits: groups, contexts, pools and layouts where it can go wrong."""

import math
import threading

import pytest
import torch

from engine.hip_decode import QuantKV, paged_decode_attention
from engine.hip_prefix import PrefixPlan, paged_prefix_attention
from prefix_cases import batch, check, expected

pytestmark = pytest.mark.gpu


def plan_of(x, **kw):
    return PrefixPlan(x.q, x.k, x.v, x.bt, x.ctx, x.groups, x.scale, x.max_ctx, quant=x.quant, **kw)


def run(x, **kw):
    return paged_prefix_attention(x.q, x.k, x.v, x.bt, x.ctx, x.groups, x.scale, x.max_ctx, quant=x.quant, **kw)


SETS = {
    "pair": ([(16, [1, 1])], []),
    "one_block": ([(64, [0, 1, 15, 16, 17])], []),
    "beams": ([(1024, [33] * 4)], []),
    "many": ([(320, [1 + 13 * (i % 9) for i in range(41)])], []),
    "groups": ([(64, [5, 70, 1]), (192, [3] * 10), (640, [300, 1]), (64, [64, 128])], [1, 17, 500]),
    "long": ([(4096, [1, 700]), (2048, [31, 32, 33])], [3000]),
    "alone": ([], [1, 16, 100, 1000]),
}


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("head_dim,heads,block", [(64, (14, 2), 16), (128, (12, 2), 16), (64, (7, 1), 32), (128, (16, 1), 64),
                                                  (64, (3, 3), 64), (128, (10, 5), 32)])
@pytest.mark.parametrize("name", SETS)
def test_batches(name, head_dim, heads, block, fmt):
    groups, alone = SETS[name]
    groups = [(max(block, p // block * block), own) for p, own in groups]
    x = batch(groups, alone, heads=heads, head_dim=head_dim, block=block, fmt=fmt, seed=len(name) + head_dim)
    check(run(x), x)
    check(run(x, host_context_lens=x.lens), x)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_groups_change_the_time_not_the_result(fmt):
    """Without groups, with smaller ones, with fewer shared tokens, with groups of one and of no tokens."""
    x = batch([(256, [20] * 9), (512, [3, 200])], [77], fmt=fmt, seed=3)
    (a, n), (b, m) = x.groups
    for groups in ([], [(a, n)], [(a[:4], n), (a[4:], n), (b, m)], [(a, 64), (b, 16)], [(a[:1], n), (b, 0), ([], 16)]):
        x.groups = groups
        check(run(x), x)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_contexts_on_the_device_decide(fmt):
    """The plan's division of the work holds for any lengths up to max_context: shorter than the prefix, zero, negative, past
    max_context (which they are clamped to), another split of the own keys than planned."""
    x = batch([(512, [300] * 6)], [700, 20], fmt=fmt, seed=5)
    plan = plan_of(x, host_context_lens=x.lens)
    full = list(x.lens)
    for ctx in ([0] * 8, [1] * 8, [511] * 8, [512] * 8, [513] * 8, [0, -7, 3, 512, 600, 100, 16, 1]):
        ctx = [min(c, f) for c, f in zip(ctx, full)]
        x.ctx.copy_(torch.tensor(ctx, dtype=torch.int32))
        check(plan(x.q, x.k, x.v), x, ctx)
    x.ctx.copy_(torch.tensor([f + 10 ** 6 if f == x.max_ctx else f for f in full], dtype=torch.int32))
    check(plan(x.q, x.k, x.v), x, full)


def test_block_ids_outside_the_pool_are_clamped():
    x = batch([(64, [20, 30])], [40], seed=6)
    x.bt[x.bt < 0] = 10 ** 9
    check(run(x), x)
    row = x.groups[0][0][0]
    x.bt[row, 4] = 2 ** 30  # the row's first own block: whatever the last block holds, the others stay right
    got, (want, tol) = run(x), expected(x, [0 if s == row else c for s, c in enumerate(x.lens)])
    others = [s for s in range(3) if s != row]
    assert ((got.double() - want).abs() <= tol)[others].all()


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.float32])
def test_strides_and_layers(fmt, scale_dtype):
    """q inside a fused projection's rows, out inside other rows, layers of larger pools, scales at odd addresses."""
    if fmt == "bf16" and scale_dtype is torch.float32:
        pytest.skip("no scales")
    x = batch([(96, [9, 40, 77])], [33], fmt=fmt, seed=8, scale_dtype=scale_dtype)
    S, Hq, D = x.q.shape
    wide = torch.randn(S, Hq + 4, D, device="cuda").bfloat16()
    wide[:, 2:2 + Hq] = x.q
    x.q = wide[:, 2:2 + Hq]
    rows = torch.full((S + 2, Hq + 3, D), 7., device="cuda").bfloat16()
    out = rows[1:1 + S, 1:1 + Hq]
    k, v = (torch.stack([torch.zeros_like(t), t, torch.zeros_like(t)]) for t in (x.k, x.v))
    quant = layers = None
    if fmt == "int8":
        def odd(t):  # [3, Hkv, N, B], one element past an aligned address
            flat = torch.zeros(3 * t.numel() + 1, dtype=t.dtype, device="cuda")
            view = flat[1:].view(3, *t.shape)
            view[1] = t
            return view

        ks, vs = odd(x.ks), odd(x.vs)
        quant, layers = QuantKV(1, ks[1], vs[1]), QuantKV(1, ks, vs)
    plan = PrefixPlan(x.q, k[1], v[1], x.bt, x.ctx, x.groups, x.scale, x.max_ctx, quant=quant)
    assert plan(x.q, k[1], v[1], out=out) is out
    check(out, x)
    rows[1:1 + S, 1:1 + Hq] = 7
    assert (rows == 7).all()
    got = plan.run_layer(1, x.q, k, v, layers)
    check(got, x)
    assert torch.equal(plan.run_layer(-2, x.q, k, v, layers), got)
    check(plan(x.q, k[1], v[1]), x)  # the plan's own scales again


def test_infinite_values():
    """Infinities in V reach the rows that see them and no others; a NaN key reaches its own rows."""
    x = batch([(128, [20, 30, 40])], [50], seed=9)
    own = x.groups[0][0][1]
    x.v[1, x.bt[own, 8], 3, 5] = math.inf          # of one member, KV head 1
    x.v[0, x.bt[own, 2], 7, 9] = -math.inf         # of the prefix, KV head 0
    got = run(x)
    check(got, x)
    assert got[own, 7:, 5].isposinf().all() and got[x.groups[0][0], :7, 9].isneginf().all()
    assert int(got.isinf().sum()) == 7 + 3 * 7
    x = batch([(128, [20, 30, 40])], [50], seed=9)
    x.k[0, x.bt[own, 9], 1, 0] = math.nan
    got = run(x)
    assert got[own, :7].isnan().all() and int(got.isnan().any(-1).any(-1).sum()) == 1


@pytest.mark.parametrize("spread", [0.001, 30.0])
def test_flat_and_peaked_softmaxes(spread):
    x = batch([(1024, [100, 3, 700])], [300], seed=10, spread=spread)
    check(run(x), x)


@pytest.mark.parametrize("up", [True, False])
def test_scores_that_rise_or_fall_along_the_keys(up):
    """The running max is raised every few tiles, or never after the first."""
    x = batch([(1024, [100, 3, 700])], [300], seed=11)
    x.k.zero_()
    for s, c in enumerate(x.lens):
        for j in range(c):
            x.k[:, x.bt[s, j // 16], j % 16, 0] = (j if up else -j) / 8
    x.q.zero_()
    x.q[:, :, 0] = 4
    check(run(x), x)


def test_agrees_with_the_decode_kernel():
    x = batch([(2048, [200, 300, 1]), (64, [1000] * 5)], [640], seed=12)
    _, tol = expected(x)
    plain = paged_decode_attention(x.q, x.k, x.v, x.bt, x.ctx, x.scale, x.max_ctx)
    assert ((run(x).double() - plain.double()).abs() <= 2 * tol).all()


def test_repeats_are_the_same_bits():
    x = batch([(640, [20] * 30), (64, [999])], [77], seed=13)
    plan = plan_of(x)
    first = plan(x.q, x.k, x.v)
    for _ in range(5):
        assert torch.equal(plan(x.q, x.k, x.v), first)
    assert torch.equal(run(x), first)


def test_captured_calls():
    """Two graphs of one plan, replayed in turn and side by side with eager work, over contexts that change between."""
    x = batch([(512, [300] * 4)], [700], seed=14)
    plan, full = plan_of(x), list(x.lens)
    plan(x.q, x.k, x.v)
    graphs = []
    for i in range(2):
        q = x.q.clone() if i == 0 else x.q.flip(0).contiguous()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = plan(q, x.k, x.v)
        graphs.append((g, out, q))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for n in (1, 600, 513, 812):
        x.ctx.copy_(torch.tensor([min(n, f) for f in full], dtype=torch.int32))
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = plan(x.q, x.k, x.v)
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], eager)
        assert torch.equal(graphs[1][1], plan(graphs[1][2], x.k, x.v))
        check(eager, x, [min(n, f) for f in full])


def test_plans_are_refused_in_a_capture():
    x = batch([(64, [9, 20])], [33], seed=19)
    run(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = x.q + 1
        with pytest.raises(ValueError, match="before the graph capture"):
            plan_of(x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, x.q + 1)


def test_streams_and_threads():
    x = batch([(512, [100] * 4)], [300], seed=15)
    plan = plan_of(x)
    qs = [torch.randn_like(x.q) for _ in range(4)]
    want = [plan(q, x.k, x.v) for q in qs]
    got = [[] for _ in qs]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(plan(qs[i], x.k, x.v))
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for w, outs in zip(want, got):
        assert len(outs) == 20 and all(torch.equal(w, o) for o in outs)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_blocks_past_four_gigabytes(fmt):
    """The same batch at the far end of a pool whose bytes and elements pass 32 bits."""
    x = batch([(128, [20, 40, 3])], [60], heads=(7, 1), seed=18, fmt=fmt)
    want = run(x)
    n, far = x.k.shape[1], (5 << 30) // (x.k.element_size() * 1024)
    k, v = (torch.empty(1, far, 16, 64, dtype=x.k.dtype, device="cuda") for _ in range(2))
    k[:, far - n:], v[:, far - n:] = x.k, x.v
    if fmt == "int8":
        ks, vs = (torch.empty(1, far, 16, dtype=torch.float16, device="cuda") for _ in range(2))
        ks[:, far - n:], vs[:, far - n:] = x.ks, x.vs
        x.quant = QuantKV(1, ks, vs)
    x.bt = torch.where(x.bt >= 0, x.bt + (far - n), x.bt)
    got = paged_prefix_attention(x.q, k, v, x.bt, x.ctx, x.groups, x.scale, x.max_ctx, quant=x.quant)
    assert torch.equal(got, want)


def test_no_sequences():
    x = batch([], [1], seed=16)
    q = x.q[:0]
    out = paged_prefix_attention(q, x.k, x.v, x.bt[:0], x.ctx[:0], [], x.scale, 1)
    assert out.shape == (0, 14, 64)


def test_refusals():
    x = batch([(64, [9, 20])], [33], seed=17)
    a = x.groups[0][0]
    for groups in ([(a, 63)], [(a, -16)], [(a, 16 * 1000)], [([a[0], a[0]], 64)], [(a, 64), (a[:1] + [2], 64)], [([0, 3], 64)],
                   [([-1, 0], 64)]):
        with pytest.raises(ValueError):
            PrefixPlan(x.q, x.k, x.v, x.bt, x.ctx, groups, x.scale, x.max_ctx)
    for kw in (dict(q=x.q.float()), dict(q=x.q[:, :13]), dict(ctx=x.ctx.long()), dict(ctx=x.ctx[:2]), dict(bt=x.bt.long()),
               dict(bt=x.bt[:, :1]), dict(max_ctx=10 ** 6), dict(k=x.k[..., :32]), dict(v=x.v.float()), dict(v=x.v[:, :3]),
               dict(quant=QuantKV(1, x.k[..., 0], x.v[..., 0])), dict(host_context_lens=[1]),
               dict(host_context_lens=[10 ** 6] * 3), dict(ctx=x.ctx.cpu())):
        a = dict(q=x.q, k=x.k, v=x.v, bt=x.bt, ctx=x.ctx, max_ctx=x.max_ctx, quant=None, host_context_lens=None)
        a.update(kw)
        with pytest.raises(ValueError):
            PrefixPlan(a["q"], a["k"], a["v"], a["bt"], a["ctx"], [], x.scale, a["max_ctx"], quant=a["quant"],
                       host_context_lens=a["host_context_lens"])
    plan = plan_of(x)
    for args, kw in (((x.q[:2], x.k, x.v), {}), ((x.q, x.k[:1], x.v), {}), ((x.q, x.k, x.v.transpose(0, 1)), {}),
                     ((x.q, x.k, x.v), dict(out=torch.empty_like(x.q).float())), ((x.q, x.k, x.v), dict(quant=QuantKV(1, x.k, x.v)))):
        with pytest.raises(ValueError):
            plan(*args, **kw)
    for scale in (0., -1., math.inf, math.nan):
        with pytest.raises(ValueError):
            paged_prefix_attention(x.q, x.k, x.v, x.bt, x.ctx, [], scale, x.max_ctx)
    check(plan(x.q, x.k, x.v), x)
