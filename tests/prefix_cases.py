"""Batches whose sequences share prefixes, and their attention in 64 bits, for the tests of the shared-prefix kernel."""

import math
from types import SimpleNamespace

import numpy as np
import torch

from engine.hip_decode import QuantKV


def batch(groups, alone, *, heads=(14, 2), head_dim=64, block=16, fmt="bf16", seed=0, shuffle=True, scale_dtype=torch.float16,
          spread=1.0):
    """groups: [(prefix tokens, own tokens of each member)], alone: contexts of the sequences that share nothing. Blocks are
    in random order, rows shuffled; what no context covers is NaN (an INT8 pool's scales)."""
    Hq, Hkv = heads
    g = torch.Generator().manual_seed(seed)
    r = np.random.RandomState(seed)
    ctx, tables, members = [], [], []
    need = sum(p // block + sum(-(-o // block) for o in own) for p, own in groups) + sum(-(-c // block) for c in alone)
    N = need + 5
    ids = iter(r.permutation(N).tolist())
    for p, own in groups:
        shared = [next(ids) for _ in range(p // block)]
        rows = []
        for o in own:
            rows.append(len(ctx))
            tables.append(shared + [next(ids) for _ in range(-(-o // block))])
            ctx.append(p + o)
        members.append((rows, p))
    for c in alone:
        tables.append([next(ids) for _ in range(-(-c // block))])
        ctx.append(c)
    S = len(ctx)
    order = r.permutation(S) if shuffle else np.arange(S)  # batch row of each
    width = max([len(t) for t in tables] + [1]) + 2
    bt = np.full((S, width), -1, dtype=np.int32)
    lens = np.zeros(S, dtype=np.int32)
    used = np.zeros((N, block), dtype=bool)
    for i, (t, c) in enumerate(zip(tables, ctx)):
        bt[order[i], :len(t)] = t
        lens[order[i]] = c
        for j in range(c):
            used[t[j // block], j % block] = True
    x = SimpleNamespace(block=block, scale=head_dim ** -0.5, fmt=fmt, lens=lens.tolist(),
                        max_ctx=max(int(lens.max(initial=1)), 1))
    x.groups = [([int(order[i]) for i in rows], p) for rows, p in members]
    x.q = (torch.randn(S, Hq, head_dim, generator=g) * spread).bfloat16().cuda()
    shape = (Hkv, N, block, head_dim)
    hole = torch.from_numpy(~used)
    if fmt == "bf16":
        x.k, x.v = (torch.randn(shape, generator=g).bfloat16() for _ in range(2))
        x.k[:, hole], x.v[:, hole] = math.nan, math.nan
        x.ks = x.vs = x.quant = None
    else:
        x.k, x.v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2))
        x.ks, x.vs = ((torch.rand(shape[:3], generator=g) * 0.02 + 0.005).to(scale_dtype) for _ in range(2))
        x.ks[:, hole], x.vs[:, hole] = math.nan, math.nan
        x.ks, x.vs = x.ks.cuda(), x.vs.cuda()
        x.quant = QuantKV(1, x.ks, x.vs)
    x.k, x.v = x.k.cuda(), x.v.cuda()
    x.bt, x.ctx = torch.from_numpy(bt).cuda(), torch.from_numpy(lens).cuda()
    return x


def expected(x, ctx=None):
    """The attention in float64 [S, Hq, D] and, element by element, how far a kernel may be from it.

    Of a row's weights: a score's fp32 sum of D products is off by at most D 2^-24 of the sum of their magnitudes (twice that
    with an INT8 scale's product), which enters the weight as a factor; the exponent's argument is rounded at 2^-24 of up to
    64 (2^-18), exp2 at 2^-22; the two bf16 terms keep 2^-15. They enter the numerator and the denominator. n keys are added
    up 16 at a time in fp32, over some parts: (n / 16 + 64) 2^-24 of the sum of p |v|, twice. The result is rounded to bf16:
    2^-8 of it."""
    S, Hq, D = x.q.shape
    Hkv = x.k.shape[0]
    G = Hq // Hkv
    out = torch.zeros(S, Hq, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for s, c in enumerate(x.lens if ctx is None else ctx):
        if c <= 0:
            continue
        ids = x.bt[s, :-(-c // x.block)].long()
        k, v = x.k[:, ids].double(), x.v[:, ids].double()
        if x.ks is not None:
            k, v = k * x.ks[:, ids].double()[..., None], v * x.vs[:, ids].double()[..., None]
        k, v = (t.reshape(Hkv, -1, D)[:, :c] for t in (k, v))
        for h in range(Hkv):
            q = x.q[s, h * G:(h + 1) * G].double()
            kt = k[h].T.contiguous()
            w = torch.softmax(q @ kt * x.scale, -1)
            o = w @ v[h]
            size = (w @ torch.where(v[h].isfinite(), v[h].abs(), 0.))
            score = 2 * D * 2 ** -24 * x.scale * (q.abs() @ kt.abs()).amax(-1, keepdim=True)
            rel = 2 * (score + 2 ** -18 + 2 ** -22 + 2 ** -15) + 2 * (c / 16 + 64) * 2 ** -24
            out[s, h * G:(h + 1) * G] = o
            tol[s, h * G:(h + 1) * G] = 2 ** -8 * o.abs() + rel * size * (1 + 2 ** -8)
    return out, tol


def check(got, x, ctx=None):
    want, tol = expected(x, ctx)
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, the worst by {float(((got - want).abs() - tol)[bad].max())}"
