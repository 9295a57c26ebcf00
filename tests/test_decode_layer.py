"""CPU tests of the decode layer's host side."""

import pytest
import torch

from decode_opt_b200 import decode_layer as dl


@pytest.mark.parametrize("requests,width,held", [(3, 5, 0), (1, 5, 2), (1, 5, 0), (3, 5, 2), (3, 5, 4), (3, 5, 5)])
def test_the_free_list_is_no_part_of_the_table(requests, width, held):
    """build_block_tables reads the one and writes the other in one launch."""
    table = torch.randperm(requests * width).to(torch.int32).view(requests, width)
    free = dl.free_list(table, held)
    assert free.dtype == torch.int32 and free.dim() == 1 and free.is_contiguous()
    assert sorted(free.tolist()) == sorted(table[:, held:].flatten().tolist())
    assert free.untyped_storage().data_ptr() != table.untyped_storage().data_ptr() or free.numel() == 0
