"""GPU tests of what the attention operators' calls do on the host: workspaces
per stream and thread."""

import threading

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import _lib

pytestmark = pytest.mark.gpu

PER_THREAD = 2      # cudaStreamPerThread: one handle, a stream for each host thread


def test_threads_on_their_per_thread_stream_have_their_own_workspaces():
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(1, 8, 128, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(200, 16, 2, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.arange(200, dtype=torch.int32, device="cuda").view(1, 200)
    lens = torch.tensor([3200], dtype=torch.int32, device="cuda")
    want = dg.paged_attention(q, k, v, table, lens)
    torch.cuda.synchronize()
    need = int(_lib.lib().dg_attention_workspace_bytes())
    grown, results = [], []

    def work():
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        dg.paged_attention(q, k, v, table, lens, out=out, stream=PER_THREAD)
        torch.cuda.synchronize()
        grown.append(torch.cuda.memory_allocated() - before)
        dg.paged_attention(q, k, v, table, lens, out=out, stream=PER_THREAD)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before == grown[-1]
        results.append(out)
    for _ in range(3):
        t = threading.Thread(target=work)
        t.start()
        t.join()
    assert len(results) == 3 and all(n >= need for n in grown), (grown, need)
    assert all(torch.equal(out, want) for out in results)


def test_a_stream_keeps_its_workspace():
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(1, 8, 128, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(8, 16, 2, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
    lens, out = torch.tensor([100], dtype=torch.int32, device="cuda"), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (None, side):
        dg.paged_attention(q, k, v, table, lens, out=out, stream=stream)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()

        def work():
            dg.paged_attention(q, k, v, table, lens, out=out, stream=stream)
        work()
        t = threading.Thread(target=work)      # the same stream, whichever thread calls
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() == before


def test_a_free_list_inside_the_block_table_is_refused():
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    new = torch.ones_like(lens)
    wide = torch.arange(30, dtype=torch.int32, device="cuda").view(3, 10)
    table = wide[:, :6]
    for free in (wide.view(-1), wide[0, 5:7], wide[1, 3:4], wide.view(-1)[8:21]):
        with pytest.raises(ValueError):
            dg.build_block_tables(lens, new, free, table, 4, 3)
    # Beside the rows it is a list like any other.
    got = dg.build_block_tables(lens, new, wide[0, 6:], table, 4, 3)
    assert table[:, 0].tolist() == [6, 7, 8] and got.cursor.tolist() == [3]
    got = dg.build_block_tables(lens, new, wide[2, 7:], table, 4, 3)
    assert table[:, 0].tolist() == [27, 28, 29] and got.slots.tolist() == [108, 112, 116]


def test_outputs_that_overlap_are_refused():
    """An output with several values in one place, or one that is moved a
    little against its own input, would be written and read in no order."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(4, 2, 64, generator=g, device="cuda").bfloat16()
    pos, rope, slots = torch.arange(4, device="cuda"), dg.rope_table(8, 64), torch.arange(4, device="cuda")
    flat = torch.zeros(5 * 128, dtype=torch.bfloat16, device="cuda")
    a, b = flat[:512].view(4, 2, 64), flat[128:].view(4, 2, 64)
    one = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device="cuda")
    flat_cache = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda").expand(2, 4, 2, 64)
    for kw in (dict(out_q=one.expand(4, 2, 64)), dict(out_k=one.expand(4, 2, 64))):
        with pytest.raises(ValueError):
            dg.rotary(q, q, pos, rope, **kw)
    for x, y in ((a, b), (b, a)):
        with pytest.raises(ValueError):
            dg.rotary(x, None, pos, rope, out_q=y)
        with pytest.raises(ValueError):
            dg.rotary(None, x, pos, rope, out_k=y)
    for caches in ((flat_cache, cache), (cache, flat_cache)):
        with pytest.raises(ValueError):
            dg.rotary_append(q, q, q, pos, slots, *caches, rope)
    with pytest.raises(ValueError):
        dg.rotary_append(q, q, q, pos, slots, cache, cache, rope)
    table, lens = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        dg.paged_attention(q, cache, cache, table, lens, out=one.expand(4, 2, 64))
    # The input itself is a fine output, and a cache that is only read may be one tensor with many names.
    want = dg.rotary(q, None, pos, rope)[0]
    assert torch.equal(dg.rotary(q, None, pos, rope, out_q=q)[0], want)
    dg.paged_attention(q, flat_cache, flat_cache, table, lens)
