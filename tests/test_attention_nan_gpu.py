"""GPU tests of paged attention where scores are NaN or -inf: the log-sum-exp
says so as the output does, wherever the token stands in the kernel's tiles."""

import pytest
import torch

from test_paged_attention_gpu import E4M3, NAN, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache,heads", [(torch.bfloat16, torch.bfloat16, 8), (torch.float16, torch.float16, 40),
                                               (torch.bfloat16, E4M3, 8)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[1], [17], [33], [129], [2049], [17] * 300, [33] * 300, [2049, 0, 5]],
                         ids=lambda n: f"{len(n)}x{n[0]}")
def test_a_nan_key_reaches_the_log_sum_exp(lens, dim, dtype, cache, heads):
    """The last token's key of kv head 0 of the first request: often the only
    live one of its tile, and the tile the only one of its warp."""
    c = Case(lens, heads, 2, dim, dtype, cache)
    want = c.run()
    n = lens[0] - 1
    page = c.table[0, n // c.page].long()
    if cache == E4M3:
        c.k_cache.view(torch.uint8)[page, n % c.page, 0, 3] = 0x7f
    else:
        c.k_cache[page, n % c.page, 0, 3] = NAN
    out, lse = c.run()
    assert out[0, :heads // 2].isnan().all() and lse[0, :heads // 2].isnan().all()
    # Everything else as before, to the bit.
    assert torch.equal(out[0, heads // 2:], want[0][0, heads // 2:])
    assert torch.equal(lse[0, heads // 2:], want[1][0, heads // 2:])
    assert torch.equal(out[1:], want[0][1:]) and torch.equal(lse[1:], want[1][1:])
