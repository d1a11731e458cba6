"""Rules on logits (engine/hip_logits.py LogitsRules, sipa_adjust_logits) against the definition in 64 bits, on the CPU
(torch operations) and on the GPU (the kernel): each rule alone and all together, types, odd vocabularies, paths of drafted
nodes, rows behind the last sequence, values that are not finite, and what is refused."""

import numpy as np
import pytest
import torch

from engine.hip_logits import LogitsRules
from tree_cases import ancestor_sets, mask_tensor, random_parents

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class Case:
    """Rules and logits of sequences with counts[s] rows each. what: the rules that are given."""

    def __init__(self, counts, vocab=1000, dtype=torch.bfloat16, device="cpu", seed=0, history=200, path=True,
                 what=("history", "prompt", "rep", "freq", "pres", "bias", "grammar"), extra=0):
        rng = np.random.RandomState(seed)
        g = torch.Generator().manual_seed(seed)
        S, R = len(counts), sum(counts) + extra
        self.counts, self.V, self.R, self.what, self.extra = counts, vocab, R, what, extra
        self.l = (torch.randn(R, vocab, generator=g) * 3).to(dtype)
        has = lambda x: x in what  # noqa: E731
        self.hist = [rng.randint(-1, vocab + 1, rng.randint(0, history + 1)) for _ in counts] if has("history") else None
        self.prompt = [int(rng.randint(0, len(h) + 1)) for h in self.hist] if has("prompt") else None
        self.rep = (rng.rand(S) + 0.6).astype(np.float32) if has("rep") else None
        self.freq = (rng.rand(S) - 0.3).astype(np.float32) if has("freq") else None
        self.pres = (rng.rand(S) - 0.3).astype(np.float32) if has("pres") else None
        self.bias = None
        if has("bias"):  # some tokens twice, some outside the vocabulary
            self.bias = [(rng.randint(-1, vocab + 1, n), rng.randn(n).astype(np.float32) * 3)
                         for n in rng.randint(0, 40, S)]
            for t, _ in self.bias:
                t[len(t) // 2:len(t) // 2 + 2] = 5
        self.tokens = rng.randint(0, vocab, R) if path else None
        self.sets = [s for n in counts for s in ancestor_sets(random_parents(n, rng))] + [set()] * extra
        self.words = -(-max(max(counts), 1) // 64)
        self.grammar = rng.randint(-(1 << 31), 1 << 31, (3, -(-vocab // 32) + 1)).astype(np.int32) if has("grammar") else None
        self.states = np.where(rng.rand(R) < 0.3, -1, rng.randint(0, 4, R)) if has("grammar") else None
        dev = lambda x, dt: None if x is None else torch.from_numpy(np.asarray(x)).to(dt).to(device)  # noqa: E731
        cat = lambda xs: np.concatenate([np.zeros(0), *xs])  # noqa: E731
        starts = lambda xs: np.concatenate([[0], np.cumsum([len(x) for x in xs])])  # noqa: E731
        kw = {}
        if self.hist is not None:
            kw |= dict(history=dev(cat(self.hist), torch.int32), history_starts=dev(starts(self.hist), torch.int64))
            kw |= dict(prompt_lens=dev(self.prompt, torch.int32))
        if self.bias is not None:
            ts = [t for t, _ in self.bias]
            kw |= dict(bias_tokens=dev(cat(ts), torch.int32), bias_starts=dev(starts(ts), torch.int32),
                       bias_values=dev(cat([x for _, x in self.bias]), torch.float32))
        self.rules = LogitsRules(vocab, S, repetition=dev(self.rep, torch.float32), frequency=dev(self.freq, torch.float32),
                                 presence=dev(self.pres, torch.float32), grammar=dev(self.grammar, torch.int32), **kw)
        self.logits = self.l.to(device)
        self.call = dict(query_starts=dev(np.concatenate([[0], np.cumsum(counts)]), torch.int32),
                         grammar_rows=dev(self.states, torch.int32))
        if path:
            self.call |= dict(tokens=dev(self.tokens, torch.int64), masks=mask_tensor(self.sets, self.words).to(device))

    def reference(self):
        """(value, tol) [R, V]. An fp32 value goes through at most a division or product, a product, two sums and the sum of
        the biases: 2^-24 each of the largest magnitude in between, and once half a step of the logits' type."""
        out = self.l.double().numpy().copy()
        size = np.abs(out)
        step = torch.finfo(self.l.dtype).eps / 2
        at = 0
        for s, n in enumerate(self.counts):
            h = self.hist[s] if self.hist is not None else np.zeros(0, dtype=int)
            k = self.prompt[s] if self.prompt is not None else 0
            for r in range(at, at + n):
                made = list(h[k:]) + ([self.tokens[at + i] for i in self.sets[r]] if self.tokens is not None else [])
                made = np.bincount([t for t in made if 0 <= t < self.V], minlength=self.V)
                seen = (made > 0) | (np.bincount([t for t in h[:k] if 0 <= t < self.V], minlength=self.V) > 0)
                l = out[r]
                if self.rep is not None:
                    rho = np.float64(self.rep[s])
                    l = np.where(seen, np.where(l > 0, l / rho, l * rho), l)
                size[r] = np.maximum(size[r], np.abs(l))
                if self.freq is not None:
                    size[r] += np.abs(self.freq[s] * made)
                    l = l - np.float64(self.freq[s]) * made
                if self.pres is not None:
                    size[r] += np.abs(self.pres[s]) * (made > 0)
                    l = l - np.float64(self.pres[s]) * (made > 0)
                if self.bias is not None:
                    for t, x in zip(*self.bias[s]):
                        if 0 <= t < self.V:
                            l[t] += np.float64(x)
                            size[r, t] += abs(x)
                if self.grammar is not None and 0 <= self.states[r] < 3:
                    v = np.arange(self.V)
                    ok = self.grammar[self.states[r]].view(np.uint32)[v // 32] >> (v % 32).astype(np.uint32) & 1
                    l = np.where(ok == 1, l, -np.inf)
                out[r] = l
            at += n
        tiny = torch.finfo(self.l.dtype).smallest_normal * step
        with np.errstate(invalid="ignore"):
            return out, 45 * 2.0 ** -24 * size + step * np.abs(out) + tiny

    def check(self, got):
        out, tol = self.reference()
        got = got.cpu().double().numpy()
        assert got.shape == out.shape
        inf = np.isinf(out)
        assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], out[inf])
        assert (np.abs(got[~inf] - out[~inf]) <= tol[~inf]).all(), np.max(np.abs(got[~inf] - out[~inf]) - tol[~inf])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 31, 1000, 8193])
def test_all_rules(device, dtype, vocab):
    c = Case([1, 4, 2, 7], vocab, dtype, device, seed=vocab)
    before = c.logits.clone()
    c.check(c.rules.apply(c.logits, **c.call))
    assert torch.equal(c.logits, before)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("what", [(), ("history",), ("history", "rep"), ("history", "prompt", "freq"), ("pres",), ("bias",),
                                  ("grammar",), ("history", "prompt", "rep", "pres")], ids=lambda w: "+".join(w) or "none")
@pytest.mark.parametrize("path", [False, True])
def test_each_rule(device, what, path):
    c = Case([3, 1, 2], 3001, torch.float32, device, seed=len(what), what=what, path=path)
    c.check(c.rules.apply(c.logits, **c.call))


@pytest.mark.parametrize("device", DEVICES)
def test_one_row_per_sequence_without_starts(device):
    c = Case([1, 1, 1, 1], 2000, torch.bfloat16, device, seed=3)
    del c.call["query_starts"]
    c.check(c.rules.apply(c.logits, **c.call))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nodes", [64, 65, 200])
def test_long_paths(device, nodes):
    c = Case([2, nodes], 500, torch.float32, device, seed=nodes)
    c.check(c.rules.apply(c.logits, **c.call))


@pytest.mark.parametrize("device", DEVICES)
def test_sequences_without_rows_and_rows_behind_the_last(device):
    c = Case([0, 2, 0, 3, 0], 777, torch.bfloat16, device, seed=4, extra=3)
    got = c.rules.apply(c.logits, **c.call)
    c.reference()
    assert torch.equal(got[5:], c.logits[5:])
    full, tol = c.reference()
    g = got.cpu().double().numpy()[:5]
    inf = np.isinf(full[:5])
    assert np.array_equal(np.isinf(g), inf) and (np.abs(g - full[:5])[~inf] <= tol[:5][~inf]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows_and_in_place(device, dtype):
    c = Case([2, 3], 1003, dtype, device, seed=5)
    wide = torch.full((5, 1100), 9.0, dtype=dtype, device=device)
    for shift in (0, 1, 3, 8):
        rows = wide[:, shift:shift + 1003]
        rows.copy_(c.logits)
        out = torch.full((5, 1021), 9.0, dtype=dtype, device=device)
        got = c.rules.apply(rows, **c.call, out=out[:, 2:1005])
        c.check(got)
        assert (out[:, :2] == 9).all() and (out[:, 1005:] == 9).all()
        assert c.rules.apply(rows, **c.call, out=rows).data_ptr() == rows.data_ptr()
        c.check(rows)
        assert (wide[:, shift + 1003:] == 9).all() and (wide[:, :shift] == 9).all()
        wide.fill_(9)


@pytest.mark.parametrize("device", DEVICES)
def test_values_that_are_not_finite(device):
    c = Case([2, 2], 64, torch.float32, device, seed=6, what=("history", "rep", "grammar"))
    c.l[:, 3], c.l[:, 4], c.l[:, 5] = float("inf"), float("-inf"), float("nan")
    c.logits.copy_(c.l)
    got = c.rules.apply(c.logits, **c.call).cpu()
    for r in range(4):
        allowed = [True] * 3
        if 0 <= c.states[r] < 3:
            allowed = [bool(c.grammar[c.states[r], 0] >> v & 1) for v in (3, 4, 5)]
        assert got[r, 3] == (float("inf") if allowed[0] else float("-inf")) and got[r, 4] == float("-inf")
        assert torch.isnan(got[r, 5]) if allowed[2] else got[r, 5] == float("-inf")


@pytest.mark.parametrize("device", DEVICES)
def test_a_grammar_that_allows_nothing_or_all(device):
    c = Case([1, 1], 100, torch.bfloat16, device, seed=7, what=("grammar",))
    c.grammar[0], c.grammar[1] = 0, -1
    c.rules.grammar.copy_(torch.from_numpy(c.grammar))
    c.call["grammar_rows"].copy_(torch.tensor([0, 1]))
    got = c.rules.apply(c.logits, **c.call)
    assert torch.isinf(got[0]).all() and (got[0] < 0).all() and torch.equal(got[1], c.logits[1])


@pytest.mark.parametrize("device", DEVICES)
def test_a_token_many_times(device):
    """Counts past 16 bits, and a bias list that names one token many times."""
    V, n = 40, 70000
    hist = torch.full((n,), 7, dtype=torch.int32, device=device)
    rules = LogitsRules(V, 1, history=hist, history_starts=torch.tensor([0, n], device=device),
                        frequency=torch.tensor([2.0 ** -10], device=device),
                        bias_tokens=torch.full((100,), 9, dtype=torch.int32, device=device),
                        bias_values=torch.full((100,), 0.5, device=device),
                        bias_starts=torch.tensor([0, 100], dtype=torch.int32, device=device))
    got = rules.apply(torch.zeros(1, V, device=device)).cpu()
    want = torch.zeros(1, V)
    want[0, 7], want[0, 9] = -n / 1024, 50.0
    assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_starts_outside_their_lists_are_clamped(device):
    # history 0 0 1 and biases of 2 and 3, with starts that point before and far behind them
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    f32 = lambda *x: torch.tensor(x, dtype=torch.float32, device=device)  # noqa: E731
    # one token a value beside the lists: entries read past them would change the second sequence's logits
    lists, biases = i32(0, 0, 1, 3, 3, 3, 3, 3), f32(4, 8, 16, 16, 16, 16)
    rules = LogitsRules(8, 2, history=lists[:3], history_starts=torch.tensor([-5, 2, 1 << 40], device=device),
                        frequency=f32(1, 1), bias_tokens=i32(2, 3, 4, 5, 6, 7)[:2], bias_values=biases[:2],
                        bias_starts=i32(-3, 1, 1 << 30))
    got = rules.apply(torch.zeros(2, 8, device=device)).cpu()
    want = torch.tensor([[-2., 0, 4, 0, 0, 0, 0, 0], [0., -1, 0, 8, 0, 0, 0, 0]])
    assert torch.equal(got, want), got


@pytest.mark.parametrize("device", DEVICES)
def test_empty_lists(device):
    z = lambda dt: torch.zeros(0, dtype=dt, device=device)  # noqa: E731
    rules = LogitsRules(10, 1, history=z(torch.int32), history_starts=torch.zeros(2, dtype=torch.int64, device=device),
                        bias_tokens=z(torch.int32), bias_values=z(torch.float32),
                        bias_starts=torch.zeros(2, dtype=torch.int32, device=device),
                        repetition=torch.full((1,), 2.0, device=device))
    l = torch.randn(1, 10, device=device)
    assert torch.equal(rules.apply(l), l)
    assert rules.apply(l[:0]).shape == (0, 10)


@pytest.mark.gpu
def test_full_vocabulary_on_the_gpu_equals_the_cpu_path():
    """151936 tokens, several workgroups a row: the kernel and the torch operations agree to the last step of the type."""
    c = Case([4, 3], 151936, torch.bfloat16, "cuda", seed=8, history=5000)
    d = Case([4, 3], 151936, torch.bfloat16, "cpu", seed=8, history=5000)
    got, want = c.rules.apply(c.logits, **c.call).cpu(), d.rules.apply(d.logits, **d.call)
    c.check(got)
    d.check(want)


@pytest.mark.gpu
def test_in_a_graph_with_new_values():
    c = Case([1, 4], 5000, torch.bfloat16, "cuda", seed=9)
    out = torch.empty_like(c.logits)
    c.rules.apply(c.logits, **c.call, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.rules.apply(c.logits, **c.call, out=out)
    for seed in (10, 11, 12):
        d = Case([1, 4], 5000, torch.bfloat16, "cuda", seed=seed, what=("rep", "freq", "grammar"))
        c.rules.repetition.copy_(d.rules.repetition)
        c.logits.copy_(d.logits)
        c.call["tokens"].copy_(d.call["tokens"])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.rules.apply(c.logits, **c.call))


def test_refusals():
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    f = lambda *x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    starts = torch.tensor([0, 2, 3])
    good = dict(history=i(1, 2, 3), history_starts=starts)
    LogitsRules(10, 2, **good)
    for kw in (dict(history=i(1)), dict(history_starts=starts), dict(prompt_lens=i(1, 1)),
               good | dict(history=torch.tensor([1])), good | dict(history_starts=starts.int()),
               good | dict(history_starts=starts[:2]), good | dict(prompt_lens=i(1)), dict(repetition=f(1)),
               dict(frequency=torch.ones(2, dtype=torch.float64)), dict(presence=f(1, 1, 1)), dict(bias_tokens=i(1)),
               dict(bias_tokens=i(1), bias_values=f(1, 2), bias_starts=i(0, 1, 1)),
               dict(bias_tokens=i(1), bias_values=f(1), bias_starts=i(0, 1)),
               dict(grammar=torch.zeros(1, 0, dtype=torch.int32)), dict(grammar=torch.zeros(1, 1)),
               dict(repetition=torch.ones(4)[::2])):
        with pytest.raises(ValueError):
            LogitsRules(10, 2, **kw)
    with pytest.raises(ValueError):
        LogitsRules(0, 1)
    r = LogitsRules(10, 2, **good, grammar=torch.zeros(1, 1, dtype=torch.int32))
    l = torch.zeros(3, 10)
    q = i(0, 1, 3)
    r.apply(l, query_starts=q)
    m = torch.zeros(3, 1, dtype=torch.int64)
    for args, kw in (((l[:, :9],), {}), ((l.double(),), {}), ((l,), {}), ((l,), dict(query_starts=q[:2])),
                     ((l,), dict(query_starts=q.long())), ((l,), dict(query_starts=q, tokens=m[:, 0])),
                     ((l,), dict(query_starts=q, masks=m)), ((l,), dict(query_starts=q, tokens=i(1, 2, 3), masks=m)),
                     ((l,), dict(query_starts=q, tokens=m[:, 0], masks=m[:2])),
                     ((l,), dict(query_starts=q, tokens=m[:, 0], masks=torch.zeros(3, 5, dtype=torch.int64))),
                     ((l,), dict(query_starts=q, grammar_rows=i(0))), ((l,), dict(query_starts=q, out=l[:2])),
                     ((l,), dict(query_starts=q, out=l.bfloat16())), ((l.t().contiguous().t(),), dict(query_starts=q))):
        with pytest.raises(ValueError):
            r.apply(*args, **kw)
    with pytest.raises(ValueError):
        LogitsRules(10, 3).apply(l, grammar_rows=i(0, 0, 0))
