"""GPU tests of dg.paged_attention against the definition in 64 bits.

Tolerance, before any run.  Let A = sum p |v| / sum p, the size of the sum
behind an output.  The result is rounded once (unit roundoff u: 2^-8 bf16,
2^-11 fp16, and to 2^-25 below fp16's normal range).  Before that: a score is
an fp32 sum of at most 256 exact products, off by at most D 2^-24 sum |q k|
scale < 2^-12.5 for these inputs; exp2 is off by 2^-22, the two-term
probabilities by 2^-16 and the fp32 sums by far less: 2^-12 A covers them.
lse: the score's error and a rounding."""

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import _lib

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn
NAN = float("nan")


class Case:
    """A cache whose every value outside the live tokens is NaN, and a table
    whose every entry outside them is far out of range."""

    def __init__(self, lens, heads, kv_heads, dim, dtype=torch.bfloat16, cache=None, page=16, window=0, cap=0.0,
                 scales=False, by_head=False, seed=0, sharp=1.0, width=None):
        cache = cache or dtype
        g = torch.Generator(device="cuda").manual_seed(seed + 131 * heads + dim)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.lens, self.window, self.cap, self.page = lens, window, cap, page
        batch, held = len(lens), [-(-n // page) for n in lens]
        pages = sum(held) + 3
        width = width or max(held) + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((batch, width), 2 ** 30, dtype=torch.int32, device="cuda")
        self.q = (rnd(batch, heads, dim) * sharp).to(dtype)
        shape = (pages, kv_heads, page, dim) if by_head else (pages, page, kv_heads, dim)
        caches = []
        for _ in range(2):
            c = torch.full(shape, NAN, device="cuda").to(cache)
            caches.append(c.transpose(1, 2) if by_head else c)
        self.k_cache, self.v_cache = caches
        self.k_scale = torch.rand(kv_heads, generator=g, device="cuda") * 0.02 + 0.01 if scales else None
        self.v_scale = torch.rand(kv_heads, generator=g, device="cuda") * 3 + 0.1 if scales else None
        self.kv, at = [], 0
        for b, n in enumerate(lens):
            self.table[b, :held[b]] = order[at:at + held[b]]
            at += held[b]
            spread = 40.0 if scales else 1.0
            rows = [(rnd(n, kv_heads, dim) * spread).to(cache) for _ in range(2)]
            tok = torch.arange(n, device="cuda")
            first = max(0, n - window) if window else 0
            where = self.table[b].long()[tok // page][first:], (tok % page)[first:]
            for c, r in zip(caches, rows):
                if cache == E4M3:
                    c.view(torch.uint8)[where] = r.view(torch.uint8)[first:]
                else:
                    c[where] = r[first:]
            self.kv.append([r[first:].double() for r in rows])
            self.table[b, :first // page] = 2 ** 30
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.scale = dim ** -0.5

    def run(self, **kw):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        kw = dict(window=self.window or None, softcap=self.cap or None, k_scale=self.k_scale, v_scale=self.v_scale,
                  return_lse=True, status=status) | kw
        out = dg.paged_attention(self.q, self.k_cache, self.v_cache, self.table, self.seq_lens, **kw)
        assert int(status) == 0, dg.status_string(int(status))
        return out

    def want(self):
        """(out, lse, A) in 64 bits."""
        batch, heads, dim = self.q.shape
        kv_heads = self.k_cache.shape[2]
        out = torch.zeros(batch, heads, dim, dtype=torch.float64, device="cuda")
        lse = torch.full((batch, heads), -torch.inf, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(out)
        group = heads // kv_heads
        for b, (k, v) in enumerate(self.kv):
            if len(k) == 0:
                continue
            if self.k_scale is not None:
                k, v = k * self.k_scale.double()[None, :, None], v * self.v_scale.double()[None, :, None]
            k, v = (x.repeat_interleave(group, 1) for x in (k, v))
            s = torch.einsum("hd,thd->ht", self.q[b].double(), k) * self.scale
            if self.cap:
                s = self.cap * torch.tanh(s / self.cap)
            p = torch.softmax(s, -1)
            lse[b] = torch.logsumexp(s, -1)
            out[b] = torch.einsum("ht,thd->hd", p, v)
            size[b] = torch.einsum("ht,thd->hd", p, v.abs())
        return out, lse, size

    def check(self, out, lse):
        want, want_lse, size = self.want()
        bound = U[out.dtype] * want.abs() + 2.0 ** -12 * size + (2.0 ** -25 if out.dtype == torch.float16 else 0.0)
        assert out.isfinite().all()
        over = ((out.double() - want).abs() - bound).max()
        assert over <= 0, float(over)
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
        far = ((lse.double() - want_lse).abs() - 2.0 ** -12 - 2.0 ** -22 * want_lse.abs())[~empty]
        assert far.numel() == 0 or far.max() <= 0, float(far.max())


LENS = [[1], [17], [0, 3, 0], [2049], [16, 32, 33, 0, 1, 255, 256, 257], [5000, 1, 0, 700]]
HEADS = [(1, 1), (8, 8), (8, 2), (8, 1), (12, 1), (32, 2), (40, 1)]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_lengths_and_groups(lens, heads, kv_heads):
    c = Case(lens, heads, kv_heads, 128)
    c.check(*c.run())


@pytest.mark.parametrize("dim", [8, 64, 72, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (20, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_dims(dim, heads, kv_heads, dtype):
    c = Case([77, 0, 1030, 16], heads, kv_heads, dim, dtype)
    c.check(*c.run())


@pytest.mark.parametrize("dim", [16, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (20, 2), (2, 2)])
@pytest.mark.parametrize("dtype,scales", [(torch.bfloat16, True), (torch.float16, True), (torch.bfloat16, False)])
def test_e4m3_cache(dim, heads, kv_heads, dtype, scales):
    c = Case([77, 0, 1030, 32, 31], heads, kv_heads, dim, dtype, E4M3, scales=scales, page=24)
    c.check(*c.run())


@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 256])
@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("cache", [torch.bfloat16, E4M3])
def test_pages_and_layouts(page, by_head, cache):
    c = Case([300, 64, 1, 129], 8, 4, 64, torch.bfloat16, cache, page=page, by_head=by_head)
    c.check(*c.run())


@pytest.mark.parametrize("window", [1, 15, 16, 100, 4096])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("cache,heads", [(torch.bfloat16, 8), (E4M3, 8), (torch.bfloat16, 24)])
def test_windows_and_caps(window, cap, cache, heads):
    """Tokens before the window lie in pages that the table no longer names."""
    c = Case([1000, 17, 0, 100, 101, 3000], heads, 2, 128, torch.bfloat16, cache, window=window, cap=cap, sharp=3.0)
    c.check(*c.run())


@pytest.mark.parametrize("batch,top", [(1, 20000), (400, 300), (148, 16), (90, 2000)])
def test_batches_cut_anywhere(batch, top):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, top + 1, (batch,), generator=g).tolist()
    c = Case(lens, 8, 2, 64, torch.float16, page=32)
    first = c.run()
    c.check(*first)
    for _ in range(3):       # tickets are left ready, and the cut sets the order of every sum
        again = c.run()
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_flat_and_sharp_scores():
    """Equal keys: every probability is 1 / n; large logits: one token takes all."""
    c = Case([5000], 4, 1, 128)
    c.k_cache[...] = torch.where(c.k_cache.isnan(), c.k_cache, torch.zeros_like(c.k_cache))
    c.kv[0][0].zero_()
    c.check(*c.run())
    c = Case([3000, 40], 4, 2, 64, torch.float16, sharp=30.0)
    c.scale = 1.0
    out, lse = c.run(scale=1.0)
    want, want_lse, size = c.want()
    # Scores reach hundreds: their fp32 rounding, 2^-24 of the sum of |q k|, allows 2^-9 of A.
    assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -9 * size + 2.0 ** -25).all()
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -20 * want_lse.abs() + 2.0 ** -9).all()


def test_quantised_result_is_the_quantisers():
    for dim, heads, kv_heads, cache in [(128, 16, 2, torch.bfloat16), (256, 4, 4, torch.bfloat16), (128, 20, 1, E4M3),
                                        (256, 3, 1, E4M3)]:
        c = Case([900, 0, 31], heads, kv_heads, dim, torch.bfloat16, cache)
        q = torch.full((3, heads * dim), 255, dtype=torch.uint8, device="cuda")
        s = torch.zeros(3, heads * dim // 128, device="cuda")
        out, lse = c.run(q_out=q, q_scales=s)
        c.check(out, lse)
        want_q, want_s = dg.quantize_activation(out.view(3, heads * dim))
        assert torch.equal(q, want_q) and torch.equal(s, want_s)


def test_strided_tensors_and_given_outputs():
    c = Case([130, 0, 999], 6, 2, 64)
    want = c.run()
    wide = torch.zeros(3, 6, 96, dtype=torch.bfloat16, device="cuda")
    wide[..., 2:66] = c.q
    c.q = wide[..., 2:66]
    full = torch.full((6, 3, 70), 7.0, dtype=torch.bfloat16, device="cuda")
    out = full.transpose(0, 1)[..., 3:67]
    got = c.run(out=out)
    assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    assert (full[..., :3] == 7).all() and (full[..., 67:] == 7).all()
    table = torch.full((3, c.table.shape[1] + 5), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, 1:1 + c.table.shape[1]] = c.table
    c.table = table[:, 1:1 + c.table.shape[1]]
    assert torch.equal(c.run()[0], want[0])


def test_offsets_past_32_bits():
    """A cache of 5 * 10^9 values (10 GB): pages at its far end."""
    pages, page, kv_heads, dim = 2 ** 18 + 2 ** 16, 16, 8, 128
    c = Case([100, 40], 8, kv_heads, dim)
    big = torch.empty(pages, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    assert big.numel() > 2 ** 32
    moved = torch.full_like(c.table, 2 ** 30)
    caches = []
    for which, small in enumerate((c.k_cache, c.v_cache)):
        at = pages - 1 - 40 * which
        for b, n in enumerate(c.lens):
            for j in range(-(-n // page)):
                big[at] = small[c.table[b, j].long()]
                if which == 0:
                    moved[b, j] = at
                at -= 1
        caches.append(big if which == 0 else big[:pages - 40])
    # Values: the same table, 40 pages further down.
    c.k_cache, c.v_cache = big[40:], big[:pages - 40]
    c.table = torch.where(moved == 2 ** 30, moved, moved - 40)
    c.check(*c.run())


def test_streams_and_graphs():
    c = Case([700, 20, 0, 3000], 8, 2, 128)
    want = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, lse = dg.paged_attention(c.q, c.k_cache, c.v_cache, c.table, c.seq_lens, return_lse=True, stream=side)
    out2 = dg.paged_attention(c.q, c.k_cache, c.v_cache, c.table, c.seq_lens, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(out2, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dg.paged_attention(c.q, c.k_cache, c.v_cache, c.table, c.seq_lens, return_lse=True)
        pdl = dg.paged_attention(c.q, c.k_cache, c.v_cache, c.table, c.seq_lens, pdl_attr=True)
    for _ in range(3):
        got[0].zero_()
        pdl.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(pdl, want[0])


def test_what_only_the_gpu_can_see_is_reported():
    c = Case([40, 33], 4, 1, 64)
    ws = dg.attention_workspace()

    def run(table, lens):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = dg.paged_attention(c.q, c.k_cache, c.v_cache, table, lens, status=status, workspace=ws)
        return out, int(status)
    # A page that is no page: its 16 tokens are left out.
    for page in (-1, c.k_cache.shape[0], 2 ** 31 - 1):
        bad = c.table.clone()
        bad[0, 1] = page
        out, code = run(bad, c.seq_lens)
        assert code == _lib.ERR_PAGE
        k, v = c.kv[0]
        keep = torch.cat([torch.arange(16), torch.arange(32, 40)]).cuda()
        p = torch.softmax(torch.einsum("hd,td->ht", c.q[0].double(), k[keep, 0]) * c.scale, -1)
        assert torch.allclose(out[0].double(), p @ v[keep, 0], atol=2.0 ** -7, rtol=2.0 ** -7)
    # Lengths out of the table's reach.
    out, code = run(c.table, torch.tensor([-5, 33], dtype=torch.int32, device="cuda"))
    assert code == _lib.ERR_SEQ_LEN and (out[0] == 0).all() and out[1].isfinite().all()
    narrow = c.table[:, :2].contiguous()
    out, code = run(narrow, torch.tensor([40, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    want, _ = run(narrow, torch.tensor([32, 32], dtype=torch.int32, device="cuda"))
    assert code == _lib.ERR_SEQ_LEN and torch.equal(out, want)
    assert int(ws[:1024].sum()) == 0


def test_infinities_and_nan_in_live_tokens_reach_the_result():
    c = Case([50, 50], 2, 2, 64, torch.float16)
    c.v_cache[c.table[0, 1].long(), 3, 0, 5] = float("inf")
    c.k_cache[c.table[1, 0].long(), 2, 1, 7] = NAN
    out = dg.paged_attention(c.q, c.k_cache, c.v_cache, c.table, c.seq_lens)
    assert out[0, 0, 5] == float("inf") and out[0, 0, :5].isfinite().all() and out[0, 1].isfinite().all()
    assert out[1, 1].isnan().all() and out[1, 0].isfinite().all()


def test_refusals():
    c = Case([40, 33], 4, 2, 64)
    ok = dict(q=c.q, k_cache=c.k_cache, v_cache=c.v_cache, block_table=c.table, seq_lens=c.seq_lens)
    f8 = c.k_cache.to(E4M3)
    two = torch.ones(2, device="cuda")
    odd = torch.zeros(2, 4, 65, dtype=torch.bfloat16, device="cuda")[..., :64]
    flat = torch.zeros(c.k_cache.numel() + 8, dtype=torch.bfloat16, device="cuda")
    off = flat[4:4 + c.k_cache.numel()].view(c.k_cache.shape)
    for bad in (dict(q=c.q.float()), dict(q=c.q.cpu()), dict(q=c.q.half()), dict(q=c.q[:1]), dict(q=c.q[:, :3]),
                dict(q=c.q[..., :32]), dict(q=odd), dict(q=c.q[:, :0]), dict(k_cache=f8), dict(k_cache=off),
                dict(v_cache=c.v_cache[:1]), dict(k_cache=c.k_cache[0]), dict(block_table=c.table.long()),
                dict(block_table=c.table[:1]), dict(block_table=c.table.cpu()), dict(block_table=c.table[:, :0]),
                dict(seq_lens=c.seq_lens.long()), dict(seq_lens=c.seq_lens[:1]), dict(window=0), dict(softcap=-1.0),
                dict(softcap=float("inf")), dict(k_scale=two), dict(k_cache=f8, v_cache=f8, k_scale=two[:1]),
                dict(out=c.q.float()), dict(out=c.q[:, :2]), dict(q_out=torch.zeros(2, 256, device="cuda")),
                dict(q_out=torch.zeros(2, 256, dtype=torch.uint8, device="cuda"), q_scales=torch.zeros(2, 2, device="cuda")),
                dict(workspace=torch.zeros(100, dtype=torch.uint8, device="cuda")), dict(status=two)):
        with pytest.raises(ValueError):
            dg.paged_attention(**{**ok, **bad})
