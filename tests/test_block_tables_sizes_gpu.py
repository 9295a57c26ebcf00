"""GPU test of dg.build_block_tables at batches around the size from which its
kernel asks for more than the ordinary 48 KiB of shared memory."""

import pytest
import torch

import decode_opt_b200 as dg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [4000, 4052, 4053, 4060, 4080, 4092, 4093, 4096, 4100, 16384])
def test_any_batch(batch):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 9, (batch,), generator=g).int()
    new = torch.randint(0, 3, (batch,), generator=g).int()
    need = (lens + new + 3) // 4 - (lens + 3) // 4
    table = torch.full((batch, 3), -7, dtype=torch.int32, device="cuda")
    free = torch.randperm(int(need.sum()) + 5, generator=g).int()
    got = dg.build_block_tables(lens.cuda(), new.cuda(), free.cuda(), table, 4, int(new.sum()))
    assert torch.equal(got.seq_lens.cpu(), lens + new)
    start = torch.cat([torch.zeros(1, dtype=torch.int32), new.cumsum(0).int()])
    assert torch.equal(got.query_start.cpu(), start) and got.cursor.item() == int(need.sum())
    row = torch.repeat_interleave(torch.arange(batch), new.long())
    assert torch.equal(got.requests.cpu(), row.int())
    position = torch.arange(len(row)) - start.long()[row] + lens.long()[row]
    assert torch.equal(got.positions.cpu(), position.int())
    want = torch.full((batch, 3), -7, dtype=torch.int32)
    taken = need.cumsum(0) - need
    for j in range(3):
        column = (lens.long() + 3) // 4 + j
        fresh = need > j
        want[fresh, column[fresh]] = free[(taken + j)[fresh].long()]
    assert torch.equal(table.cpu(), want)
