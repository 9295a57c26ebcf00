"""GPU tests of one decode layer run on two streams at once, and as a captured
graph beside them: every call's attention has tickets and shares of its own."""

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import decode_layer as dl

pytestmark = pytest.mark.gpu

SHAPE = dl.LayerShape(1024, 16, 2, 128)
BATCH, PAGE, CONTEXT = 4, 16, 3001


def _state(seed):
    """Lengths that give every request's items to several CTAs."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = CONTEXT // PAGE + 1
    cache = dl.PagedCache(SHAPE, BATCH * width, PAGE)
    for c in (cache.k, cache.v):
        c.copy_(torch.randn(c.shape, generator=g, device="cuda"))
    table = torch.randperm(BATCH * width, generator=g, device="cuda").to(torch.int32).view(BATCH, width)
    lens = torch.full((BATCH,), CONTEXT, dtype=torch.int32, device="cuda") - torch.arange(BATCH, device="cuda").int() * 100
    step = dg.build_block_tables(lens, torch.ones_like(lens), torch.empty(0, dtype=torch.int32, device="cuda"), table,
                                 PAGE, BATCH)
    x = torch.randn(BATCH, SHAPE.hidden, generator=g, device="cuda").bfloat16()
    return x, step, table, cache


def test_workspaces_are_not_shared(monkeypatch):
    """Whatever the layer hands to paged_attention differs from stream to
    stream; nothing, where that call finds its own."""
    layer, rope = dl.random_layer(SHAPE, BATCH), dg.rope_table(CONTEXT + 8, 128)
    given, real = [], dg.paged_attention
    monkeypatch.setattr(dg, "paged_attention", lambda *a, workspace=None, **kw: given.append(workspace) or real(
        *a, workspace=workspace, **kw))
    a = _state(1)
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            layer.step(*a, rope)
        stream.synchronize()
    assert len(given) == 2 and (given[0] is None or given[0] is not given[1])
    mine = dg.attention_workspace()
    layer.step(*a, rope, workspace=mine)
    assert given[2] is mine


def test_two_streams_and_a_graph():
    layer, rope = dl.random_layer(SHAPE, BATCH), dg.rope_table(CONTEXT + 8, 128)
    states = [_state(s) for s in (1, 2, 3)]
    want = [layer.step(*s, rope) for s in states]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[2]):
        captured = layer.step(*states[2], rope)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(100):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(layer.step(*states[i], rope))
        with torch.cuda.stream(streams[2]):
            graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    assert torch.equal(captured, want[2])
