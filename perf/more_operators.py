"""What the operators of decoding with shared prefixes are measured on: the calls of a program that decodes several
beams, or several requests, over one stored prompt, each through the public entry point that it would use, with inputs
made from a seed, the work that the call cannot do without, and the result in 64 bits.

A case is a dict of plain values. Kinds:

  attend  one layer's decode attention of sequences whose tables begin with the same blocks, the shared keys read once
          for all of them (engine.hip_prefix.PrefixPlan, built once per forward and called once per layer)
  select  the best continuations of every request's beams over beams and vocabulary, by log-probability
          (engine.hip_beam.beam_select)
  copy    the states of beams that go on from another beam: the tokens of a block that is not full yet, copied in all
          layers (engine.hip_beam.copy_blocks; full blocks are shared)

With `own` false, run() computes the same in elementary torch operations in 32 bits; scores of continuations, which
decide between tokens, in 64.

Sizes: the two attention shapes are those of engine/config.py; batches and contexts are the benchmark's or generic; the
vocabulary is the configurations' or a generic odd one.
"""

import math
import random
import sys
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda"
SHAPES = {"0.5b": dict(layers=24, hq=14, hkv=2, d=64), "1.5b": dict(layers=28, hq=12, hkv=2, d=128)}
VOCAB = 151936


# ---- the cases -----------------------------------------------------------------------------------------------------


def listed():
    return [
        # Four beams of one chat turn: latency is all there is.
        dict(name="attend_beams", kind="attend", shape="0.5b", fmt="bf16", block=16, groups=1, members=4, prefix=1024,
             suffix=33, ragged=False, alone=0),
        # A batch of requests with eight beams each, some tokens into their answers.
        dict(name="attend_beam_batch", kind="attend", shape="0.5b", fmt="bf16", block=16, groups=8, members=8,
             prefix=4096, suffix=300, ragged=True, alone=0),
        # A full batch behind one system prompt, every request with a conversation of its own.
        dict(name="attend_system", kind="attend", shape="1.5b", fmt="bf16", block=16, groups=1, members=256,
             prefix=2048, suffix=600, ragged=True, alone=0),
        # INT8 pools: several long prompts with many answers each, among requests that share nothing.
        dict(name="attend_int8", kind="attend", shape="1.5b", fmt="int8", block=16, groups=4, members=15, prefix=4096,
             suffix=500, ragged=True, alone=4),
        # Many short answers to questions on two long documents, on 32-token blocks: the most work a step asks for.
        dict(name="attend_document", kind="attend", shape="0.5b", fmt="bf16", block=32, groups=2, members=37,
             prefix=30016, suffix=100, ragged=True, alone=0),
        # The next tokens of one request's four beams.
        dict(name="select_one", kind="select", dtype="bfloat16", vocab=VOCAB, groups=1, beams=4, candidates=8,
             masked=False),
        # The first step of a batch, one row a request, 16-bit floats of an odd vocabulary.
        dict(name="select_first", kind="select", dtype="float16", vocab=50257, groups=32, beams=1, candidates=10,
             masked=False),
        # A smaller, odd vocabulary in 32 bits, most of it forbidden by a grammar.
        dict(name="select_f32", kind="select", dtype="float32", vocab=32003, groups=24, beams=3, candidates=6,
             masked=True),
        # Every beam of a full batch.
        dict(name="select_batch", kind="select", dtype="bfloat16", vocab=VOCAB, groups=64, beams=8, candidates=16,
             masked=False),
        # One request's beams, of which two are replaced; a batch of requests on an INT8 cache.
        dict(name="copy_one", kind="copy", shape="0.5b", fmt="bf16", copies=2, tokens=9),
        dict(name="copy_batch", kind="copy", shape="1.5b", fmt="int8", copies=384, tokens=15),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: 1 to 32 prefixes of up to 32768 tokens, groups of 2 to 256 sequences, 1 to 4096 tokens of their
    own; vocabularies from 1000, 1 to 16 beams, 1 to 32 candidates; 1 to 512 copies."""
    kind = rng.choice(["attend"] * 3 + ["select"] * 2 + ["copy"])
    if kind == "attend":
        shape = rng.choice(["0.5b", "1.5b"])
        width = SHAPES[shape]["hq"] * SHAPES[shape]["d"]
        block = rng.choice([16, 16, 32, 64])
        groups = _log(rng, 1, 32)
        members = _log(rng, 2, max(2, min(256, 400 // groups)))
        alone = rng.choice([0, 0, rng.randint(1, 9)])
        seqs = groups * members + alone
        most = 2_000_000_000 // (2 * width * seqs)  # keys a sequence, so that no case costs more than the largest
        prefix = max(1, _log(rng, block, max(block, min(32768, most, 150000 // groups))) // block) * block
        suffix = _log(rng, 1, max(1, min(4096, most, 100000 // seqs)))
        return dict(kind=kind, shape=shape, fmt=rng.choice(["bf16", "bf16", "int8"]), block=block, groups=groups,
                    members=members, prefix=prefix, suffix=suffix, ragged=rng.random() < 0.7, alone=alone)
    if kind == "select":
        beams = _log(rng, 1, 16)
        return dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                    vocab=rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), groups=_log(rng, 1, 256 // beams), beams=beams,
                    candidates=rng.randint(1, 32), masked=rng.random() < 0.3)
    return dict(kind=kind, shape=rng.choice(["0.5b", "1.5b"]), fmt=rng.choice(["bf16", "int8"]),
                copies=_log(rng, 1, 384), tokens=rng.randint(1, 15))


# ---- sizes of a case -----------------------------------------------------------------------------------------------


def _own_tokens(case):
    """Tokens of its own of each sequence, the same for the same case: the groups' members one group after the other,
    then the sequences that share nothing (their whole context)."""
    r = random.Random(case["groups"] * 1009 + case["members"] * 31 + case["prefix"] + case["suffix"])

    def vary(n):
        return max(1, round(n * r.uniform(0.3, 1.7))) if case["ragged"] else n

    return ([vary(case["suffix"]) for _ in range(case["groups"] * case["members"])],
            [vary(case["prefix"] + case["suffix"]) for _ in range(case["alone"])])


def _copy_tokens(case):
    """Tokens of each copied block: up to the case's, at least half of them."""
    r = random.Random(case["copies"] * 31 + case["tokens"])
    return [r.randint((case["tokens"] + 1) // 2, case["tokens"]) for _ in range(case["copies"])]


# ---- inputs --------------------------------------------------------------------------------------------------------


def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed(seed * 1000 + salt)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.bfloat16)


def _quantize(x):
    """INT8 codes of x and one fp16 scale per row, absmax / 127."""
    s = (x.abs().amax(-1).float() / 127).half()
    q = (x.float() / s.float().clamp_min(1e-30)[..., None]).round().clamp(-127, 127)
    return q.to(torch.int8), s


def _attend_inputs(case, seed):
    s, B = SHAPES[case["shape"]], case["block"]
    mine, alone = _own_tokens(case)
    shared = case["prefix"] // B
    per = [-(-n // B) for n in mine]
    per_alone = [-(-n // B) for n in alone]
    n = case["groups"] * shared + sum(per) + sum(per_alone)
    n += n // 8 + 8
    r = np.random.RandomState(seed % (1 << 31))
    ids = r.permutation(n).astype(np.int32)  # a pool that has served for a while
    S = len(mine) + len(alone)
    bt = np.full((S, max([shared + p for p in per] + per_alone)), -1, dtype=np.int32)
    ctx = np.zeros(S, dtype=np.int64)
    # beams of a request stand together; other sequences are in the order of their arrival
    order = r.permutation(S) if case["ragged"] else np.arange(S)
    prefixes = ids[:case["groups"] * shared].reshape(case["groups"], shared)
    at = case["groups"] * shared
    groups = []
    for g in range(case["groups"]):
        rows = order[g * case["members"]:(g + 1) * case["members"]]
        for j, row in enumerate(rows):
            i = g * case["members"] + j
            bt[row, :shared] = prefixes[g]
            bt[row, shared:shared + per[i]] = ids[at:at + per[i]]
            at += per[i]
            ctx[row] = case["prefix"] + mine[i]
        groups.append((sorted(rows.tolist()), case["prefix"]))
    for i, row in enumerate(order[len(mine):]):
        bt[row, :per_alone[i]] = ids[at:at + per_alone[i]]
        at += per_alone[i]
        ctx[row] = alone[i]
    g = _gen(seed)
    k, v = _randn(g, s["hkv"], n, B, s["d"]), _randn(g, s["hkv"], n, B, s["d"])
    x = SimpleNamespace(scale=s["d"] ** -0.5, block=B, ks=None, vs=None, groups=groups, max_ctx=int(ctx.max()))
    if case["fmt"] == "int8":
        (k, x.ks), (v, x.vs) = _quantize(k), _quantize(v)
    x.k, x.v = k, v
    x.q = _randn(g, S, s["hq"], s["d"])
    x.bt = torch.from_numpy(bt).to(DEV)
    x.ctx = torch.from_numpy(ctx.astype(np.int32)).to(DEV)
    return x


def _select_inputs(case, seed):
    R, V = case["groups"] * case["beams"], case["vocab"]
    g = _gen(seed)
    x = SimpleNamespace(V=V, beams=case["beams"], candidates=case["candidates"])
    x.logits = torch.randn(R, V, generator=g, device=DEV) * 3
    if case["masked"]:  # a grammar leaves a few tokens, another beam is free
        few = torch.rand(R, V, generator=g, device=DEV) < 40 / V
        few[:, torch.randint(0, V, (1,), generator=g, device=DEV)] = True
        few |= torch.rand(R, 1, generator=g, device=DEV) < 0.3
        x.logits.masked_fill_(~few, -math.inf)
    x.logits = x.logits.to(getattr(torch, case["dtype"]))
    # log-probabilities of a few tokens so far, nearer to each other than their sum is to zero
    x.scores = -30 * torch.rand(case["groups"], 1, generator=g, device=DEV) - 4 * torch.rand(
        case["groups"], case["beams"], generator=g, device=DEV)
    x.scores = x.scores.reshape(R)
    return x


def _copy_inputs(case, seed):
    s, B = SHAPES[case["shape"]], 16
    n = 2 * case["copies"] + case["copies"] // 4 + 8
    ids = np.random.RandomState(seed % (1 << 31)).permutation(n)[:2 * case["copies"]].reshape(2, -1).tolist()
    g = _gen(seed)
    shape = (s["layers"], s["hkv"], n, B, s["d"])
    if case["fmt"] == "int8":
        pools = [torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
        pools += [torch.rand(shape[:-1], generator=g, device=DEV).half() for _ in range(2)]
    else:
        pools = [_randn(g, *shape), _randn(g, *shape)]
    return SimpleNamespace(pools=tuple(pools), copies=list(zip(*ids, _copy_tokens(case))))


_INPUTS = dict(attend=_attend_inputs, select=_select_inputs, copy=_copy_inputs)


def prepare(case, seed):
    x = _INPUTS[case["kind"]](case, seed)
    x.kind = case["kind"]
    if own:
        path = str(Path.cwd() / "small-inference_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        if x.kind == "attend":  # what a serving program keeps over a forward: the attention's plan
            from engine.hip_decode import QuantKV
            from engine.hip_prefix import PrefixPlan

            quant = None if x.ks is None else QuantKV(1, x.ks, x.vs)
            x.plan = PrefixPlan(x.q, x.k, x.v, x.bt, x.ctx, x.groups, x.scale, x.max_ctx, quant=quant)
    return x


# ---- one pass ------------------------------------------------------------------------------------------------------


def run(x):
    if not own:
        return _PLAIN[x.kind](x)
    if x.kind == "attend":
        return x.plan(x.q, x.k, x.v)
    from engine.hip_beam import beam_select, copy_blocks

    if x.kind == "select":
        return tuple(beam_select(x.logits, x.scores, x.beams, x.candidates))
    copy_blocks(x.pools, x.copies)
    return x.pools


def _plain_attend(x):
    S, Hq, D = x.q.shape
    H = x.k.shape[0]
    G, C = Hq // H, x.bt.shape[1] * x.block
    ids = x.bt.clamp_min(0).long()

    def gather(pool, scale):
        t = pool[:, ids].float()  # [H, S, blocks, B, D]
        if scale is not None:
            t = t * scale[:, ids].float()[..., None]
        return t.reshape(H * S, C, D)

    q = x.q.float().view(S, H, G, D).transpose(0, 1).reshape(H * S, G, D)
    scores = torch.bmm(q, gather(x.k, x.ks).transpose(1, 2).contiguous()) * x.scale
    hidden = torch.arange(C, device=DEV)[None, :] >= x.ctx[:, None]
    scores = scores.view(H, S, G, C).masked_fill(hidden[None, :, None, :], -math.inf).view(H * S, G, C)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.bmm(p, gather(x.v, x.vs)) / p.sum(-1, keepdim=True)
    return o.view(H, S, G, D).transpose(0, 1).reshape(S, Hq, D).to(x.q.dtype)


def _plain_select(x):
    R, V = x.logits.shape
    K, N = x.beams, x.candidates
    l, top = [], x.logits.float().amax(-1).double()
    for a in range(0, R, 64):  # some rows at a time: 64 bits of every logit need room
        p = torch.exp(x.logits[a:a + 64].double() - top[a:a + 64, None])
        l.append(top[a:a + 64] + torch.log(p.sum(-1)))
    value, token = torch.sort(x.logits.float(), dim=-1, descending=True, stable=True)  # ties: the lower token first
    n = min(N, V)
    value, token = value[:, :n], token[:, :n]
    score = x.scores.double()[:, None] + (value.double() - torch.cat(l)[:, None])
    score = score.view(-1, K * n)
    score, at = torch.sort(score, dim=-1, descending=True, stable=True)  # ties: the lower beam first
    score, at = score[:, :N], at[:, :N]
    none = score == -math.inf
    beam = torch.where(none, -1, at // n)
    token = torch.where(none, -1, torch.gather(token.reshape(-1, K * n), 1, at))
    return score.float(), beam, token


def _plain_copy(x):
    src, dst, tokens = (torch.tensor(c, device=DEV) for c in zip(*x.copies))
    live = torch.arange(16, device=DEV)[None, :] < tokens[:, None]
    pair, at = live.nonzero(as_tuple=True)
    for pool in x.pools:
        pool[:, :, dst[pair], at] = pool[:, :, src[pair], at]
    return x.pools


_PLAIN = dict(attend=_plain_attend, select=_plain_select, copy=_plain_copy)


# ---- the work of a pass --------------------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "attend":
        s = SHAPES[case["shape"]]
        mine, alone = _own_tokens(case)
        S = len(mine) + len(alone)
        per = 2 * s["hkv"] * (s["d"] * 2 if case["fmt"] == "bf16" else s["d"] + 2)
        stored = case["groups"] * case["prefix"] + sum(mine) + sum(alone)  # the shared tokens once
        pairs = len(mine) * case["prefix"] + sum(mine) + sum(alone)
        return {"bytes": stored * per + S * s["hq"] * s["d"] * 4, "flops": 4 * pairs * s["hq"] * s["d"]}
    if kind == "select":
        R, size = case["groups"] * case["beams"], 4 if case["dtype"] == "float32" else 2
        return {"bytes": R * (case["vocab"] * size + 4) + case["groups"] * case["candidates"] * 20,
                "flops": 4.0 * R * case["vocab"]}
    s = SHAPES[case["shape"]]
    row = 2 * s["d"] if case["fmt"] == "bf16" else s["d"] + 2
    return {"bytes": 2 * sum(_copy_tokens(case)) * 2 * s["layers"] * s["hkv"] * row, "flops": 0}


# ---- the result in 64 bits -----------------------------------------------------------------------------------------


def exact(case, seed):
    """The definition, one sequence (attention) or one row (selection) after another, in float64. Copies: None."""
    if case["kind"] == "attend":
        return _exact_attend(case, _attend_inputs(case, seed))
    if case["kind"] == "select":
        return _exact_select(case, _select_inputs(case, seed))
    return None


def _exact_attend(case, x):
    s = SHAPES[case["shape"]]
    G = s["hq"] // s["hkv"]
    out = torch.empty(x.q.shape, dtype=torch.float64, device=DEV)
    for i, c in enumerate(x.ctx.tolist()):
        ids = x.bt[i, :-(-c // x.block)].long()
        k, v = x.k[:, ids].double(), x.v[:, ids].double()
        if x.ks is not None:
            k, v = k * x.ks[:, ids].double()[..., None], v * x.vs[:, ids].double()[..., None]
        k, v = (t.reshape(s["hkv"], -1, s["d"])[:, :c] for t in (k, v))
        for h in range(s["hkv"]):
            z = (x.q[i, h * G:(h + 1) * G].double() @ k[h].T.contiguous()) * x.scale
            out[i, h * G:(h + 1) * G] = torch.softmax(z, -1) @ v[h]
    return out


def _exact_select(case, x):
    G, K, N, V = case["groups"], case["beams"], case["candidates"], case["vocab"]
    logits, cum = x.logits.float().cpu().numpy(), x.scores.double().cpu().numpy()
    score, beam, token = np.full((G, N), -np.inf), np.full((G, N), -1), np.full((G, N), -1)
    for g in range(G):
        found = []
        for b in range(K):
            l = logits[g * K + b].astype(np.float64)
            top = l.max()
            total = cum[g * K + b] - (top + np.log(np.exp(l - top).sum()))
            least = np.partition(l, V - min(N, V))[V - min(N, V)]
            found += [(-(total + l[t]), b, t) for t in np.flatnonzero((l >= least) & (l > -np.inf))]
        for i, (z, b, t) in enumerate(sorted(found)[:N]):
            score[g, i], beam[g, i], token[g, i] = -z, b, t
    return tuple(torch.from_numpy(t).to(DEV) for t in (score, beam, token))
