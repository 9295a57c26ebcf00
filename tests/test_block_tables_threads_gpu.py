"""GPU test of dg_build_block_tables from two host threads at once: what one
call sets for its kernel (its shared memory grows with the batch) must not
refuse the other's launch."""

import ctypes
import threading

import pytest
import torch

from decode_opt_b200 import _lib

pytestmark = pytest.mark.gpu


def _call(batch, stream):
    ints = torch.zeros(8 * batch + 64, dtype=torch.int32, device="cuda")
    ints[:batch] = 3
    ints[batch:2 * batch] = 1
    part = [ints[i * batch:].data_ptr() for i in range(8)]
    slots = torch.empty(batch, dtype=torch.int64, device="cuda")
    a = _lib.DgBlockTables(batch=batch, page_size=16, table_width=1, num_tokens=batch, free_count=0, table_stride=1,
                           context_lens=part[0], new_lens=part[1], block_table=part[2], seq_lens=part[3],
                           positions=part[4], requests=part[5], query_start=part[6], cursor_out=part[7] + 4 * 32,
                           slots=slots.data_ptr())
    return a, (ints, slots, stream)


def test_two_threads_with_batches_of_their_own():
    L, codes = _lib.lib(), {}
    batches = (16384, 5000)
    calls = [_call(b, torch.cuda.Stream()) for b in batches]
    torch.cuda.synchronize()
    gate = threading.Barrier(2)

    def work(i):
        a, (_, _, stream) = calls[i]
        gate.wait()
        bad = 0
        for _ in range(4000):
            bad += L.dg_build_block_tables(ctypes.byref(a), stream.cuda_stream, 0) != 0
        codes[i] = bad
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == {0: 0, 1: 0}
    for (a, (ints, slots, _)), b in zip(calls, batches):
        assert (ints[3 * b:4 * b] == 4).all() and (slots == 3).all()
