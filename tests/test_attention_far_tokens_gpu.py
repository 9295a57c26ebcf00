"""GPU tests of tokens without weight in paged attention: scores far below the
largest, or -inf."""

import pytest
import torch

from test_paged_attention_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,dim", [(4, 64), (4, 128), (20, 128), (4, 256)])
def test_far_tokens_have_no_weight(dtype, heads, dim):
    """One token whose value is 0 holds all the weight (a head that looks at
    nothing); the 100,000 others, at exp(-50), have values of 1.  200 requests
    share the pages, so that a warp has thousands of tokens in one sum.  The
    bound is check()'s: fp16's smallest rounding, the weighted sizes being
    1e5 * exp(-50)."""
    n = 100000
    c = Case([n], heads, 1, dim, dtype)
    keys, values = c.kv[0]
    keys.zero_()
    keys[5] = 1.0
    c.q.fill_(50.0 / dim ** 0.5)
    values.fill_(1.0)
    values[5] = 0.0
    tok = torch.arange(n, device="cuda")
    page, inside = c.table[0].long()[tok // c.page], tok % c.page
    c.k_cache[page, inside], c.v_cache[page, inside] = keys.to(dtype), values.to(dtype)
    c.q, c.table, c.seq_lens = (x.repeat_interleave(200, 0) for x in (c.q, c.table, c.seq_lens))
    out, lse = c.run()
    assert (out == out[:1]).all() and (lse == lse[:1]).all()
    c.q = c.q[:1]
    c.check(out[:1], lse[:1])


@pytest.mark.parametrize("lens", [[1], [33], [2049], [33] * 300], ids=lambda n: f"{len(n)}x{n[0]}")
def test_scores_of_minus_infinity(lens):
    """Some: they have no weight.  All: the sum is 0, its logarithm -inf, and
    the output 0 / 0, as the definition's."""
    c = Case(lens, 4, 2, 64, torch.float16)
    c.q[0] = c.q[0].abs() + 0.5
    n = lens[0]
    tok = torch.arange(n, device="cuda")
    page, inside = c.table[0].long()[tok // c.page], tok % c.page
    if n > 1:
        c.k_cache[page[n // 2:], inside[n // 2:], 0] = -torch.inf
        c.kv[0][0][n // 2:, 0] = -torch.inf
        c.check(*c.run())
    c.k_cache[page, inside, 0] = -torch.inf
    out, lse = c.run()
    assert out[0, :2].isnan().all() and (lse[0, :2] == -torch.inf).all()
    assert out[0, 2:].isfinite().all() and lse[0, 2:].isfinite().all()
