"""GPU tests of capped logits over the caps' whole range.

Tolerances, before any run.  Against the definition: as in
test_paged_attention_gpu.py.  The cap by itself: the same scores, to the bit,
go through the call with and without the cap, and the difference of the two
log-sum-exps is compared with that of the definition.  A capped score is off by
2^-21 of itself (a tanh of 32 bits) and the roundings of a division and two
products; each exponential by 2^-22 of itself and 2^-24 of its argument's parts,
each logarithm and its sum by 2^-22 of lse.  The sums' weights add up to 1, so
that 2^-20 of the largest score and 2^-20 * (1 + |lse|) cover the difference."""

import pytest
import torch

from test_paged_attention_gpu import E4M3, Case

pytestmark = pytest.mark.gpu

CAPS = [0.01, 1.0, 5.0, 30.0, 1.0e3, 1.0e4, 1.0e5, 1.0e8, 1.0e20, 3.0e38]
SHAPES = [(torch.bfloat16, torch.bfloat16, 8, 128), (torch.float16, torch.float16, 24, 64),
          (torch.bfloat16, E4M3, 24, 128), (torch.float16, torch.float16, 8, 256)]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,cache,heads,dim", SHAPES)
def test_any_cap(cap, dtype, cache, heads, dim):
    c = Case([1000, 17, 0, 1, 300], heads, 2, dim, dtype, cache, sharp=3.0)
    _, plain = c.run()
    _, want_plain, _ = c.want()
    c.cap = cap
    out, lse = c.run()
    c.check(out, lse)
    _, want, _ = c.want()
    top = torch.stack([torch.einsum("hd,thd->ht", c.q[b].double(), k.repeat_interleave(heads // 2, 1)).abs().amax(1)
                       if len(k) else torch.zeros(heads, dtype=torch.float64, device="cuda")
                       for b, (k, _) in enumerate(c.kv)]) * c.scale
    far = ((lse.double() - plain.double()) - (want - want_plain)).abs()
    live = torch.isfinite(want)
    bound = 2.0 ** -20 * (top + 1 + want_plain.abs() + want.abs())
    assert (far - bound)[live].max() <= 0, float((far / bound)[live].max())


@pytest.mark.parametrize("cap", [1.0, 30.0])
def test_scores_far_past_the_cap(cap):
    """Saturated on either side: all tokens of a sign weigh the same."""
    c = Case([700], 2, 1, 64, torch.float16, sharp=200.0)
    c.cap = cap
    c.check(*c.run())
