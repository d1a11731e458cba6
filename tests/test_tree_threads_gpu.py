"""One TreePlan and one LogitsRules called by several threads at once, each on a stream of its own: the library is called
without the interpreter's lock, and every call has to launch its own arguments. The library is wrapped so that a call waits
a moment before it reads them: calls that were not kept apart would meet there."""

import threading
import time

import pytest
import torch

from engine import _hip
from engine.hip_logits import LogitsRules
from engine.hip_tree import TreePlan
from tree_cases import Case

pytestmark = pytest.mark.gpu


class Slow:
    """The library, with a pause at the start of every call."""

    def __init__(self, lib):
        self._lib = lib

    def __getattr__(self, name):
        f = getattr(self._lib, name)

        def call(*args):
            time.sleep(0.003)
            return f(*args)

        return call


def together(calls):
    """Each of calls, 10 times, in a thread and on a stream of its own; their results."""
    results, errors = [[] for _ in calls], []
    gate = threading.Barrier(len(calls))
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    gate.wait(timeout=20)
                    results[i].append(calls[i]())
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # a thread's exception ends its test
            errors.append(e)
            gate.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    return results


@pytest.mark.parametrize("int8", [False, True])
def test_a_plan_in_several_threads(int8):
    c = Case([(900, 6), (30, 9)], (14, 2, 64), int8=int8, seed=51)
    plan = TreePlan(c.q, c.k, c.v, c.bt, c.ctx, c.qs, c.masks, c.scale, c.max_ctx, c.max_nodes, quant=c.quant(), num_splits=3)
    qs = [c.q * (i + 1) for i in range(4)]
    k, v, scales = torch.stack([c.k, c.k]), torch.stack([c.v, c.v]), c.quant()
    if int8:
        scales = type(scales)(1, torch.stack([c.ks, c.ks]), torch.stack([c.vs, c.vs]))
    want = [plan(q, c.k, c.v) for q in qs]
    plan._lib = Slow(plan._lib)
    calls = [lambda q=q: plan(q, c.k, c.v) for q in qs[:2]] + [lambda q=q: plan.run_layer(1, q, k, v, scales) for q in qs[2:]]
    for got, w in zip(together(calls), want):
        assert all(torch.equal(x, w) for x in got)


def test_rules_in_several_threads(monkeypatch):
    V = 5000
    rules = LogitsRules(V, 3, frequency=torch.tensor([1.0, 2.0, 3.0], device="cuda"),
                        history=torch.arange(3000, dtype=torch.int32, device="cuda"),
                        history_starts=torch.tensor([0, 10, 2000, 3000], device="cuda"))
    logits = [torch.randn(3, V, device="cuda").to(t) for t in (torch.bfloat16, torch.float32, torch.float16, torch.float32)]
    want = [rules.apply(l) for l in logits]
    lib = Slow(_hip.lib())
    monkeypatch.setattr(_hip, "lib", lambda: lib)
    for got, w in zip(together([lambda l=l: rules.apply(l) for l in logits]), want):
        assert all(torch.equal(x, w) for x in got)
