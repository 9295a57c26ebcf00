"""GPU tests of the attention half of a decode layer: several steps through
block tables, products, rotary, cache and attention together."""

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import decode_layer as dl

pytestmark = pytest.mark.gpu


def _turned(x, positions, theta=10000.0):
    x = x.double()
    d = x.shape[-1]
    angle = positions.double()[:, None] * theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("shape,batch,window", [
    (dl.LayerShape(1024, 16, 2, 128), 5, None), (dl.LayerShape(1024, 8, 8, 128), 17, 9),
    (dl.LayerShape(512, 16, 4, 64), 1, None), (dl.LayerShape(768, 24, 1, 128), 128, None)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_steps(shape, batch, window, e4m3):
    """Each step equals its operators called one by one, bit for bit, and its
    attention equals the definition in 64 bits over everything that the steps
    so far have cached.

    Tolerance of that: the cache holds k and v rounded as the definition's are
    here (they are read back from it), q is the rotated bf16 q itself; what is
    left is paged_attention's own: one bf16 rounding (2^-8 of the value) and
    2^-12 of the sum of the values' sizes."""
    if window is not None:
        shape = dl.LayerShape(shape.hidden, shape.heads, shape.kv_heads, shape.head_dim, window=window)
    page, steps = 4, 11
    layer = dl.random_layer(shape, batch, seed=batch)
    g = torch.Generator(device="cuda").manual_seed(9)
    width = -(-steps // page)
    free = torch.randperm(batch * width, generator=g, device="cuda").to(torch.int32)
    block_table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    scales = [torch.full((shape.kv_heads,), 0.02, device="cuda") if e4m3 else None for _ in range(2)]
    kind = torch.float8_e4m3fn if e4m3 else torch.bfloat16
    cache, other = (dl.PagedCache(shape, batch * width, page, kind, *scales) for _ in range(2))
    table = dg.rope_table(64, shape.head_dim)
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    new = torch.ones_like(lens)
    cursor = torch.zeros(1, dtype=torch.int32, device="cuda")
    h, hk, d = shape.heads, shape.kv_heads, shape.head_dim
    for n in range(1, steps + 1):
        x = torch.randn(batch, shape.hidden, generator=g, device="cuda").bfloat16()
        t = dg.build_block_tables(lens, new, free, block_table, page, batch, cursor=cursor)
        y = layer.step(x, t, block_table, cache, table)
        # One by one.
        act, s = dg.quantize_activation(x)
        qkv = dg.fp8_decode_gemm(act, s, layer.w_qkv, layer.qkv_scales, config=layer.qkv_config, n=shape.qkv_width)
        qkv = qkv.view(batch, h + 2 * hk, d)
        q = dg.rotary_append(qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:], t.positions, t.slots, other.k, other.v,
                             table, k_scale=scales[0], v_scale=scales[1])
        bits = torch.uint8 if e4m3 else torch.int16
        assert torch.equal(other.k.view(bits), cache.k.view(bits)) and torch.equal(other.v.view(bits),
                                                                                   cache.v.view(bits))
        out = dg.paged_attention(q, other.k, other.v, block_table, t.seq_lens, window=window, k_scale=scales[0],
                                 v_scale=scales[1])
        act, s = dg.quantize_activation(out.view(batch, h * d))
        z = dg.fp8_decode_gemm(act, s, layer.w_out, layer.out_scales, config=layer.out_config, n=shape.hidden)
        assert torch.equal(y, z) and y.isfinite().all()
        # The definition.
        assert t.seq_lens.tolist() == [n] * batch and t.positions.tolist() == [n - 1] * batch
        want_q = _turned(qkv[:, :h], t.positions)
        assert ((q.double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 1e-5).all()
        first = max(0, n - window) if window else 0
        tok = torch.arange(first, n, device="cuda")
        rows = block_table.long()[:, tok // page] * page + tok % page                       # [B, tokens]
        k, v = (c.float().view(-1, hk, d)[rows].double() for c in (cache.k, cache.v))
        if e4m3:
            k, v = k * scales[0].double()[:, None], v * scales[1].double()[:, None]
        k, v = (c.repeat_interleave(h // hk, 2) for c in (k, v))
        p = torch.softmax(torch.einsum("bhd,bthd->bht", q.double(), k) * d ** -0.5, -1)
        want, size = torch.einsum("bht,bthd->bhd", p, v), torch.einsum("bht,bthd->bhd", p, v.abs())
        assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * size).all()
        lens.copy_(t.seq_lens)
        cursor.copy_(t.cursor)
    assert len(set(block_table.flatten().tolist())) == batch * width


def test_main_runs(capsys):
    assert dl.main(["--requests", "3", "--context", "50", "--steps", "2", "--hidden", "512", "--heads", "4", "--kv-heads",
                    "2", "--page-size", "16", "--e4m3-cache"]) == 0
    assert "us a step" in capsys.readouterr().out


def test_refusals():
    with pytest.raises(ValueError):
        dl.random_layer(dl.LayerShape(500, 4, 2, 128), 1)
    w = torch.zeros(1024, 512, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError):
        dl.DecodeAttention(dl.LayerShape(512, 4, 2, 128), w[:128], None, w, None, 1)
