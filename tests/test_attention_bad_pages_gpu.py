"""GPU tests of paged attention where no page of a request is one of the
cache's, as after build_block_tables ran out of free pages: its tokens are left
out, so that it has none -- 0, log-sum-exp -inf, the smallest scale."""

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import _lib
from test_paged_attention_gpu import E4M3, Case

pytestmark = pytest.mark.gpu

# One short request; short ones (a warp each); items of one CTA and of several.
LENS = {"one": [5], "short": [20, 0, 31] * 130, "items": [480, 600, 512] * 60, "split": [20000, 40, 3000]}


@pytest.mark.parametrize("which", LENS)
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (128, 20, 1), (256, 4, 1), (256, 24, 2), (64, 6, 6)])
@pytest.mark.parametrize("cache", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("page", [32, 24])
def test_nothing_but_bad_pages(which, dim, heads, kv_heads, cache, page):
    lens = LENS[which]
    c = Case(lens, heads, kv_heads, dim, torch.bfloat16, cache, page=page, scales=cache == E4M3)
    c.check(*c.run())
    bad = torch.arange(0, len(lens), 2, device="cuda")
    good = torch.arange(1, len(lens), 2, device="cuda")
    want, want_lse = c.run()
    c.table[bad] = -1
    c.table[bad[::2]] = c.k_cache.shape[0]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = {}
    if dim % 128 == 0:
        kw = dict(q_out=torch.full((len(lens), heads * dim), 255, dtype=torch.uint8, device="cuda"),
                  q_scales=torch.full((len(lens), heads * dim // 128), -1.0, device="cuda"))
    out, lse = c.run(status=status, **kw)
    assert int(status) == _lib.ERR_PAGE
    assert (out[bad] == 0).all() and (lse[bad] == -torch.inf).all()
    assert torch.equal(out[good], want[good]) and torch.equal(lse[good], want_lse[good])
    if kw:
        want_q, want_s = dg.quantize_activation(out.view(len(lens), heads * dim))
        assert torch.equal(kw["q_out"], want_q) and torch.equal(kw["q_scales"], want_s)
