"""GPU tests of what autograd sees of the attention operators."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import decode_opt_b200 as dg
import decode_opt_b200.attention as attention

pytestmark = pytest.mark.gpu


def _rotary_inputs(dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(5, 4, 32, generator=g, device="cuda").to(dtype)
    k = torch.randn(5, 2, 32, generator=g, device="cuda").to(dtype)
    return q, k, torch.arange(3, 8, device="cuda"), dg.rope_table(16, 16)


def _attention_inputs():
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(2, 4, 128, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(4, 8, 2, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    return q, k, v, table, torch.tensor([5, 16], dtype=torch.int32, device="cuda")


def test_rotary_forward_mode():
    """The map is linear: its derivative along a tangent is itself."""
    q, k, pos, table = _rotary_inputs()
    tq, tk = torch.randn_like(q), torch.randn_like(k)
    for pairing in ("half", "adjacent"):
        for inverse in (False, True):
            kw = dict(pairing=pairing, inverse=inverse)
            want, want_t = dg.rotary(q, k, pos, table, **kw), dg.rotary(tq, tk, pos, table, **kw)
            with fwd.dual_level():
                got = dg.rotary(fwd.make_dual(q, tq), fwd.make_dual(k, tk), pos, table, **kw)
                for x, y, t in zip(got, want, want_t):
                    x = fwd.unpack_dual(x)
                    assert torch.equal(x.primal, y) and torch.equal(x.tangent, t)
                # One of the two, alone and beside the other; a broadcast tangent.
                one = fwd.make_dual(q, torch.ones((), device="cuda").expand_as(q))
                ones = dg.rotary(torch.ones_like(q), None, pos, table, **kw)[0]
                got = dg.rotary(one, k, pos, table, **kw)
                assert torch.equal(fwd.unpack_dual(got[0]).tangent, ones)
                assert fwd.unpack_dual(got[1]).tangent is None and torch.equal(got[1], want[1])
                got = dg.rotary(one, None, pos, table, **kw)
                assert torch.equal(fwd.unpack_dual(got[0]).tangent, ones) and got[1] is None
                with pytest.raises(ValueError):
                    dg.rotary(one, None, pos, table, out_q=torch.empty_like(q), **kw)


def test_forward_over_reverse():
    """A dual that also wants a gradient: both derivatives."""
    q, k, pos, table = _rotary_inputs()
    t = torch.randn_like(q)
    leaf = q.clone().requires_grad_()
    with fwd.dual_level():
        y = dg.rotary(fwd.make_dual(leaf, t), None, pos, table)[0]
        assert torch.equal(fwd.unpack_dual(y).tangent, dg.rotary(t, None, pos, table)[0])
        (g,) = torch.autograd.grad(y.sum(), leaf)
        g = fwd.unpack_dual(g).primal
    assert torch.equal(g, dg.rotary(torch.ones_like(q), None, pos, table, inverse=True)[0])


def test_forward_mode_is_refused_where_there_is_no_derivative():
    q, kc, vc, table, lens = _attention_inputs()
    x, k, pos, rope = _rotary_inputs(torch.bfloat16)
    cache = torch.zeros(2, 4, 2, 32, device="cuda", dtype=torch.bfloat16)
    with fwd.dual_level():
        with pytest.raises(ValueError):
            dg.paged_attention(fwd.make_dual(q, torch.ones_like(q)), kc, vc, table, lens)
        with pytest.raises(ValueError):
            dg.paged_attention(q, kc, fwd.make_dual(vc, torch.ones_like(vc)), table, lens)
        with pytest.raises(ValueError):
            dg.rotary_append(x, k, fwd.make_dual(k, torch.ones_like(k)), pos, torch.arange(5, device="cuda"), cache,
                             cache.clone(), rope)
        dg.paged_attention(q, kc, vc, table, lens)


def test_tensors_that_want_a_gradient_and_get_none_are_refused():
    q, kc, vc, table, lens = _attention_inputs()
    f8 = kc.to(torch.float8_e4m3fn)
    scale = torch.ones(2, device="cuda")
    wants = lambda t: t.clone().requires_grad_()  # noqa: E731
    for args, kw in (((wants(q), kc, vc), {}), ((q, wants(kc), vc), {}), ((q, kc, wants(vc)), {}),
                     ((q, f8, f8), dict(k_scale=wants(scale))), ((q, f8, f8), dict(v_scale=wants(scale))),
                     ((q, kc, vc), dict(out=wants(q))),
                     ((q, kc, vc), dict(q_out=torch.empty(2, 512, dtype=torch.uint8, device="cuda"),
                                        q_scales=wants(torch.ones(2, 4, device="cuda"))))):
        with pytest.raises(ValueError):
            dg.paged_attention(*args, table, lens, **kw)
        with torch.no_grad():
            dg.paged_attention(*args, table, lens, **kw)
    x, k, pos, rope = _rotary_inputs(torch.bfloat16)
    slots = torch.arange(5, device="cuda")
    cache = torch.zeros(2, 4, 2, 32, device="cuda", dtype=torch.bfloat16)
    c8, ones = cache.to(torch.float8_e4m3fn), torch.ones(2, device="cuda")
    for args, kw in (((wants(x), k, k, pos, slots, cache, cache.clone(), rope), {}),
                     ((x, k, k, pos, slots, wants(cache), cache.clone(), rope), {}),
                     ((x, k, k, pos, slots, cache, wants(cache), rope), {}),
                     ((x, k, k, pos, slots, cache, cache.clone(), wants(rope)), {}),
                     ((x, k, k, pos, slots, c8, c8.clone(), rope), dict(k_scale=wants(ones))),
                     ((x, k, k, pos, slots, cache, cache.clone(), rope), dict(out_q=wants(x)))):
        with pytest.raises(ValueError):
            dg.rotary_append(*args, **kw)
        with torch.no_grad():
            dg.rotary_append(*args, **kw)
    for args, kw in (((x, k, pos, wants(rope)), {}), ((wants(x), k, pos, wants(rope)), {}),
                     ((x, k, pos, rope), dict(out_q=wants(x))), ((x, k, pos, rope), dict(out_k=wants(k)))):
        with pytest.raises(ValueError):
            dg.rotary(*args, **kw)


def test_written_tensors_have_a_new_version():
    q, kc, vc, table, lens = _attention_inputs()
    x, k, pos, rope = _rotary_inputs(torch.bfloat16)
    slots = torch.arange(5, device="cuda")

    def bumped(call, *tensors):
        before = [t._version for t in tensors]
        call()
        return [t._version > b for t, b in zip(tensors, before)]
    caches = [torch.zeros(2, 4, 2, 32, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    assert all(bumped(lambda: dg.rotary_append(x, k, k, pos, slots, *caches, rope, out_q=x), x, *caches))
    assert all(bumped(lambda: dg.rotary(x, k, pos, rope, out_q=x, out_k=k), x, k))
    out, bits, s = q.clone(), torch.empty(2, 512, dtype=torch.uint8, device="cuda"), torch.empty(2, 4, device="cuda")
    assert all(bumped(lambda: dg.paged_attention(q, kc, vc, table, lens, out=out, q_out=bits, q_scales=s), out, bits, s))
    new, free = torch.ones_like(lens), torch.arange(4, 8, dtype=torch.int32, device="cuda")
    wide = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    step = dg.build_block_tables(lens, new, free, wide, 8, 2)
    parts = (step.seq_lens, step.query_start, step.slots, step.positions, step.requests, step.cursor)
    assert all(bumped(lambda: dg.build_block_tables(lens, new, free, wide, 8, 2, out=step), wide, *parts))
    # Inputs keep theirs.
    assert not any(bumped(lambda: dg.paged_attention(q, kc, vc, table, lens), q, kc, vc, table, lens))
    # What it is for: autograd notices that what it saved was overwritten.
    w = torch.ones_like(q, requires_grad=True)
    saved = q.clone()
    loss = (w * saved).sum()
    dg.paged_attention(q, kc, vc, table, lens, out=saved)
    with pytest.raises(RuntimeError):
        loss.backward()
    # Inference tensors have no versions, and are served as before.
    with torch.inference_mode():
        there = torch.empty_like(q)
    dg.paged_attention(q, kc, vc, table, lens, out=there)
    assert torch.equal(there, out)


def test_tracing_is_refused():
    """A trace would keep the results of this one call as constants."""
    q, kc, vc, table, lens = _attention_inputs()
    x, k, pos, rope = _rotary_inputs(torch.bfloat16)
    slots = torch.arange(5, device="cuda")
    cache = torch.zeros(2, 4, 2, 32, device="cuda", dtype=torch.bfloat16)
    free = torch.arange(4, 8, dtype=torch.int32, device="cuda")
    for f, given in ((lambda q: dg.paged_attention(q, kc, vc, table, lens), q),
                     (lambda q: dg.rotary(q, k, pos, rope)[0], x),
                     (lambda q: dg.rotary_append(q, k, k, pos, slots, cache, cache.clone(), rope), x),
                     (lambda n: dg.build_block_tables(lens, n, free, table.clone(), 8, 2).slots, torch.ones_like(lens))):
        f(given)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(f, (given,), check_trace=False)


class _Spy:
    """The extension module, with rotary's calls noted."""

    def __init__(self, real, calls):
        self.real, self.calls = real, calls

    def __getattr__(self, name):
        return getattr(self.real, name)

    def rotary(self, *args):
        self.calls.append(args)
        return self.real.rotary(*args)


def test_backward_turns_back_what_is_wanted_only(monkeypatch):
    q, k, pos, table = _rotary_inputs()
    calls = []
    monkeypatch.setattr(attention, "_host", _Spy(attention._host, calls))
    for wq, wk in ((True, False), (False, True), (True, True)):
        a, b = q.clone().requires_grad_(wq), k.clone().requires_grad_(wk)
        y, z = dg.rotary(a, b, pos, table)
        assert (y.requires_grad, z.requires_grad) == (wq, wk)
        del calls[:]
        (sum(t.sum() for t in (y, z) if t.requires_grad)).backward()
        assert [(c[0] is not None, c[1] is not None) for c in calls] == [(wq, wk)]
        for t, g in ((a, q), (b, k)):
            if t.requires_grad:
                ones = torch.ones_like(g)
                assert torch.equal(t.grad, dg.rotary(ones, None, pos, table, inverse=True)[0])
    # Both could have one, and only one result is used.
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    y, _ = dg.rotary(a, b, pos, table)
    del calls[:]
    ga, gb = torch.autograd.grad(y.sum(), (a, b), allow_unused=True)
    assert len(calls) == 1 and calls[0][1] is None and gb is None and ga is not None
