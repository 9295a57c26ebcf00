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
