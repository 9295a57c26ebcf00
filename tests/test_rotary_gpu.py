"""GPU tests of dg.rotary and dg.rotary_append against the definition in 64
bits.

Tolerance, before any run: the kernel rounds its result once to the output
type (unit roundoff u: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32) after two fp32
products, one sum and a table rounded to fp32: at most 4 * 2^-24 * (|x| + |y|)
before that rounding.  fp16 results below its normal range are rounded to
2^-25."""

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import _lib

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
THETA, MAX_POSITION = 10000.0, 70000


def _axes(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def _turned(x, positions, rot, sections, interleaved, pairing, inverse):
    """(the definition in 64 bits, |x| + |y| of each value's pair)."""
    x = x.double().cpu()
    axes = torch.tensor(_axes(sections or (rot // 2,), interleaved))
    p = positions.cpu().double()
    p = p[None].expand(int(axes.max()) + 1, -1) if p.dim() == 1 else p
    angle = p[axes].T * THETA ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if inverse else 1)
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if pairing == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    out, size = x.clone(), x.abs()
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return out, size


def _near(got, want, size, dtype):
    bound = U[dtype] * want.abs() + 4 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert got.shape == want.shape
    over = (got.double().cpu() - want).abs() - bound
    assert (over <= 0).all(), float(over.max())


def _positions(tokens, axes, dtype, g):
    shape = (tokens,) if axes == 0 else (axes, tokens)
    return torch.randint(0, MAX_POSITION, shape, generator=g, device="cuda").to(dtype)


CASES = [  # tokens, heads, kv_heads, dim, rot, sections, interleaved, pairing, axes of positions (0: one row)
    (1, 1, 1, 64, 64, None, False, "half", 0),
    (5, 8, 2, 128, 128, (16, 24, 24), False, "half", 3),
    (33, 3, 1, 128, 64, (12, 10, 10), True, "adjacent", 3),
    (7, 4, 4, 80, 40, None, False, "half", 1),
    (9, 2, 1, 96, 96, (48,), False, "adjacent", 1),
    (300, 5, 5, 64, 32, (4, 6, 6), True, "half", 3),
    (4, 2, 2, 10, 6, (1, 2), False, "half", 2),
    (3, 2, 1, 7, 2, None, False, "adjacent", 0),
    (601, 64, 8, 128, 128, None, False, "half", 0),
    (2, 1, 1, 512, 512, (64, 64, 64, 64), True, "half", 4),
    (1000, 1, 1, 16, 16, (0, 4, 4), False, "half", 3),
    (5, 2, 2, 256, 192, (32, 32, 32), False, "half", 0),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotary_matches_the_definition(case, dtype, inverse):
    tokens, heads, kv_heads, dim, rot, sections, interleaved, pairing, axes = case
    g = torch.Generator(device="cuda").manual_seed(tokens * 7 + dim)
    q = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(dtype)
    k = torch.randn(tokens, kv_heads, dim, generator=g, device="cuda").to(dtype)
    positions = _positions(tokens, axes, torch.int64 if tokens % 2 else torch.int32, g)
    table = dg.rope_table(MAX_POSITION, rot, THETA)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(sections=sections, interleaved=interleaved, pairing=pairing, inverse=inverse, status=status)
    got = dg.rotary(q, k, positions, table, **kw)
    for x, y in zip((q, k), got):
        _near(y, *_turned(x, positions, rot, sections, interleaved, pairing, inverse), dtype)
        assert torch.equal(y[..., rot:], x[..., rot:])
    # One of the two alone, and into the input: the same bits.
    assert torch.equal(dg.rotary(q, None, positions, table, **kw)[0], got[0])
    assert torch.equal(dg.rotary(None, k, positions, table, **kw)[1], got[1])
    q2, k2 = q.clone(), k.clone()
    assert dg.rotary(q2, k2, positions, table, out_q=q2, out_k=k2, **kw)[0] is q2
    assert torch.equal(q2, got[0]) and torch.equal(k2, got[1])
    assert int(status) == 0


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_rotary_on_slices_of_a_projection(offset):
    """Strided inputs and outputs, whatever their alignment: the bits of the
    contiguous call."""
    tokens, heads, kv_heads, dim = 21, 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(tokens, (heads + kv_heads) * dim + 8, generator=g, device="cuda").bfloat16()
    q = wide[:, offset:offset + heads * dim].unflatten(1, (heads, dim))
    k = wide[:, offset + heads * dim:offset + (heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    positions, table = _positions(tokens, 0, torch.int64, g), dg.rope_table(MAX_POSITION, dim, THETA)
    want = dg.rotary(q.contiguous(), k.contiguous(), positions, table)
    out = torch.zeros(heads, tokens, dim + 8, device="cuda", dtype=torch.bfloat16)
    out_q = out.transpose(0, 1)[:, :, offset:offset + dim]
    got = dg.rotary(q, k, positions, table, out_q=out_q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rest = torch.ones(dim + 8, dtype=torch.bool)
    rest[offset:offset + dim] = False
    assert (out[..., rest.cuda()] == 0).all()


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_gradient_is_the_formulas_and_the_differences(pairing):
    tokens, heads, dim, rot = 6, 2, 24, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(tokens, heads, dim, generator=g, device="cuda").requires_grad_()
    k = torch.randn(tokens, 1, dim, generator=g, device="cuda").requires_grad_()
    positions, table = _positions(tokens, 3, torch.int64, g), dg.rope_table(MAX_POSITION, rot, THETA)
    kw = dict(sections=(2, 3, 3), interleaved=True, pairing=pairing)
    wq, wk = torch.randn_like(q), torch.randn_like(k)

    def loss(q, k):
        a, b = dg.rotary(q, k, positions, table, **kw)
        return (a.double() * wq).sum() + (b.double() * wk).sum()
    gq, gk = torch.autograd.grad(loss(q, k), (q, k))
    for x, got in ((wq, gq), (wk, gk)):
        _near(got, *_turned(x, positions, rot, (2, 3, 3), True, pairing, True), torch.float32)
    # The map is linear: a difference of any width is its derivative, up to
    # the rounding of two results (2^-23 of values below 8) over the width.
    for t, h, d in [(0, 0, 0), (3, 1, 7), (5, 0, 8), (2, 1, 15), (4, 0, 23)]:
        step = torch.zeros_like(q)
        step[t, h, d] = 1.0
        with torch.no_grad():
            diff = (loss(q + step, k) - loss(q - step, k)) / 2
        assert abs(float(diff - gq[t, h, d])) < 1e-4
    # A gradient for one of the two, and a broadcast gradient.
    (only,) = torch.autograd.grad(dg.rotary(q, k.detach(), positions, table, **kw)[0].sum(), q)
    _near(only, *_turned(torch.ones_like(q), positions, rot, (2, 3, 3), True, pairing, True), torch.float32)
    (alone,) = torch.autograd.grad(dg.rotary(q, None, positions, table, **kw)[0].sum(), q)
    assert torch.equal(alone, only)


def _cache(pages, page, heads, dim, dtype, by_head, g):
    shape = (pages, heads, page, dim) if by_head else (pages, page, heads, dim)
    c = torch.randn(shape, generator=g, device="cuda").to(dtype)
    return c.transpose(1, 2) if by_head else c


def _bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x.view(torch.int16)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,page,by_head", [
    (1, 1, 1, 64, 64, 16, False), (8, 64, 8, 128, 128, 16, False), (77, 6, 2, 80, 40, 24, True),
    (400, 4, 4, 96, 96, 1, False), (1500, 2, 1, 10, 6, 64, True), (5, 3, 3, 256, 128, 32, True)])
@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.uint8)])
def test_append_matches_the_definition(tokens, heads, kv_heads, dim, rot, page, by_head, dtype, cache):
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    real = torch.float8_e4m3fn if cache == torch.uint8 else cache
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g, device="cuda").to(dtype)
    q = qkv[:, :heads * dim].unflatten(1, (heads, dim))
    k = qkv[:, heads * dim:(heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    v = qkv[:, (heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim))
    pages = tokens // page + 3
    caches = [_cache(pages, page, kv_heads, dim, real, by_head, g) for _ in range(2)]
    before = [c.clone() for c in caches]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[::5] = -1
    positions, table = _positions(tokens, 0, torch.int64, g), dg.rope_table(MAX_POSITION, rot, THETA)
    e4m3 = real == torch.float8_e4m3fn
    scales = [torch.rand(kv_heads, generator=g, device="cuda") * 0.05 + 0.004 if e4m3 else None for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    given = [c.view(torch.uint8) if cache == torch.uint8 else c for c in caches]
    got = dg.rotary_append(q, k, v, positions, slots, *given, table, k_scale=scales[0], v_scale=scales[1],
                           status=status)
    assert int(status) == 0
    assert torch.equal(got, dg.rotary(q, None, positions, table)[0])
    live = slots >= 0
    page_of, inside = slots[live] // page, slots[live] % page
    want_k, size_k = _turned(k, positions, rot, None, False, "half", False)
    for c, old, want, size, scale in zip(caches, before, (want_k, v.double().cpu()), (size_k, v.double().abs().cpu()),
                                         scales):
        rows = c[page_of, inside] if not e4m3 else c.view(torch.uint8)[page_of, inside].view(real)
        if e4m3:
            want, size = want / scale.double().cpu()[None, :, None], size / scale.double().cpu()[None, :, None]
            want = want[live.cpu()].clamp(-448, 448)
            # u = 2^-4, subnormals rounded to 2^-10
            err = (rows.float().double().cpu() - want).abs()
            assert (err <= 2.0 ** -4 * want.abs() + 2.0 ** -10 + 8 * 2.0 ** -24 * size[live.cpu()]).all()
        else:
            _near(rows, want[live.cpu()], size[live.cpu()], dtype)
        untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        untouched[page_of, inside] = False
        assert torch.equal(_bits(c)[untouched], _bits(old)[untouched])


def test_append_saturates_and_keeps_nan():
    q = torch.zeros(1, 1, 16, device="cuda", dtype=torch.bfloat16)
    v = q.clone()
    v[0, 0, :5] = torch.tensor([1e4, -1e4, float("inf"), float("nan"), 3.0], device="cuda")
    kc = torch.zeros(1, 1, 1, 16, device="cuda", dtype=torch.float8_e4m3fn)
    vc = kc.clone()
    table = dg.rope_table(4, 16)
    slot = torch.zeros(1, dtype=torch.int64, device="cuda")
    dg.rotary_append(q, q.clone(), v, slot, slot, kc, vc, table)
    row = vc.float().flatten()[:5].tolist()
    assert row[:3] == [448.0, -448.0, 448.0] and row[3] != row[3] and row[4] == 3.0


def test_positions_and_slots_outside_are_reported():
    q = torch.randn(3, 2, 16, device="cuda").bfloat16()
    table = dg.rope_table(10, 16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, _ = dg.rotary(q, None, torch.tensor([9, 10, -1], device="cuda"), table, status=status)
    assert int(status) == _lib.ERR_POSITION
    assert out[0].isfinite().all() and out[1:].isnan().all()
    status.zero_()
    kc = torch.zeros(2, 4, 2, 16, device="cuda", dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    slots = torch.tensor([7, 8, 2 ** 40], device="cuda")
    dg.rotary_append(q, q.clone(), q.clone(), torch.zeros(3, dtype=torch.int64, device="cuda"), slots, kc, vc, table,
                     status=status)
    assert int(status) == _lib.ERR_SLOT
    assert torch.equal(vc[1, 3], q[0]) and int((vc != 0).any(-1).any(-1).sum()) == 1


def test_refusals():
    q = torch.zeros(4, 2, 16, device="cuda", dtype=torch.bfloat16)
    pos, table = torch.zeros(4, dtype=torch.int64, device="cuda"), dg.rope_table(8, 16)
    cache = torch.zeros(2, 4, 2, 16, device="cuda", dtype=torch.bfloat16)
    f8 = cache.to(torch.float8_e4m3fn)
    scale = torch.ones(2, device="cuda")
    ok = dict(q=q, k=q, positions=pos, table=table)
    for bad in (dict(q=q.cpu()), dict(q=q.double()), dict(k=q.half()), dict(k=q[:3]), dict(q=None, k=None),
                dict(positions=pos[:3]), dict(positions=pos.float()), dict(positions=pos.expand(3, 4)),
                dict(sections=(4, 2)), dict(sections=(2, 2, 2, 1, 1)), dict(sections=(9, -1)), dict(pairing="both"),
                dict(table=dg.rope_table(8, 32)), dict(table=table.double()), dict(table=table.cpu()),
                dict(out_q=q[:, :1]), dict(out_q=q.float()), dict(status=pos), dict(q=q[..., ::2])):
        with pytest.raises(ValueError):
            dg.rotary(**{**ok, **bad})
    ok = dict(q=q, k=q, v=q, positions=pos, slots=pos, k_cache=cache, v_cache=cache, table=table)
    for bad in (dict(v=None), dict(v=q[:, :1]), dict(slots=pos.int()), dict(slots=pos[:3]), dict(k_cache=f8),
                dict(k_cache=cache.half(), v_cache=cache.half()), dict(k_cache=cache[:, :, :1]), dict(k_scale=scale),
                dict(k_cache=f8, v_cache=f8, v_scale=scale[:1]), dict(v_cache=cache[:1])):
        with pytest.raises(ValueError):
            dg.rotary_append(**{**ok, **bad})
