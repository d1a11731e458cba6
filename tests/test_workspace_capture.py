"""Split workspaces made inside a graph capture: only the graph's replays fill them with zeros, so that no call outside of it,
and no other graph, may count in them."""

import types

import pytest
import torch

from engine import _hip, hip_decode


def test_a_workspace_made_in_a_capture_is_the_captures_own(monkeypatch):
    """On the CPU, with the capture's id as the library would give it."""
    capture = 0
    zeros = torch.zeros
    monkeypatch.setattr(_hip, "lib", lambda: types.SimpleNamespace(sipa_capture_id=lambda stream: capture))
    monkeypatch.setattr(torch, "zeros", lambda n, dtype, device: zeros(n, dtype=dtype))
    for name in ("_workspaces", "_captured"):
        monkeypatch.setattr(hip_decode, name, {}, raising=False)
    dev, take = torch.device("cuda", 0), hip_decode.reserve_workspace
    capture = 5
    first = take(dev, 77, 100)
    assert take(dev, 77, 1 << 20) is first  # every layer of the capture
    larger = take(dev, 77, 3 << 20)
    assert larger.numel() == 3 << 20 and take(dev, 77, 100) is larger
    capture = 6
    other = take(dev, 77, 100)
    assert other is not first and other is not larger
    capture = 0
    eager = take(dev, 77, 100)
    assert eager is not first and eager is not larger and eager is not other and take(dev, 77, 100) is eager
    capture = 7
    assert take(dev, 77, 100) is eager  # one that was there serves captures too
    assert take(dev, 77, 2 << 20) is not eager
    capture = 0
    assert take(dev, 77, 100) is eager


@pytest.mark.gpu
def test_captures_without_a_call_before(monkeypatch):
    """Decodes of several splits captured on a stream without a workspace, two graphs; then eager ones on that stream before any
    replay, and replays of both graphs side by side: all as the eager call elsewhere."""
    for name in ("_workspaces", "_captured"):
        monkeypatch.setattr(hip_decode, name, {})
    S, H, N, ctx = 4, 2, 300, 1100
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(S, 14, 64, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(H, N, 16, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    bt = torch.randperm(N, generator=g, device="cuda")[:S * 69].view(S, 69).int()
    lens = torch.full((S,), ctx, dtype=torch.int32, device="cuda")

    def call():
        return hip_decode.paged_decode_attention(q, k, v, bt, lens, 0.125, ctx, num_splits=6)

    want = call()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = [call() for _ in range(2)]
        graphs.append((graph, out))
    assert list(hip_decode._captured) == [(0, s.cuda_stream)]
    with torch.cuda.stream(s):
        eager = [call() for _ in range(2)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in eager)
    others = [torch.cuda.Stream() for _ in graphs]
    for seed in range(4):
        q.copy_(torch.randn(S, 14, 64, generator=g, device="cuda"))
        want = call()
        torch.cuda.synchronize()
        for (graph, out), t in zip(graphs, others):
            for x in out:
                x.zero_()
        torch.cuda.synchronize()
        for (graph, _), t in zip(graphs, others):
            with torch.cuda.stream(t):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for _, out in graphs for x in out)
