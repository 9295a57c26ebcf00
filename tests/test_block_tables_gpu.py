"""GPU tests of dg.build_block_tables against a loop over the requests (whole
numbers: exact)."""

import pytest
import torch

import decode_opt_b200 as dg
from decode_opt_b200 import _lib

pytestmark = pytest.mark.gpu


def _ceil(a, b):
    return -(-a // b)


def _reference(context, new, free, table, page, num_tokens, cursor=0):
    table = [row[:] for row in table]
    start, slots, positions, requests = [0], [], [], []
    for b, (c, n) in enumerate(zip(context, new)):
        for j in range(_ceil(c, page), _ceil(c + n, page)):
            table[b][j] = free[cursor]
            cursor += 1
        for p in range(c, c + n):
            slots.append(table[b][p // page] * page + p % page)
            positions.append(p)
            requests.append(b)
        start.append(start[-1] + n)
    pad = num_tokens - len(slots)
    return {"table": table, "seq_lens": [c + n for c, n in zip(context, new)], "query_start": start,
            "slots": slots + [-1] * pad, "positions": positions + [0] * pad, "requests": requests + [-1] * pad,
            "cursor": [cursor]}


def _inputs(context, new, page, width, seed=0, spare=5):
    g = torch.Generator().manual_seed(seed)
    need = sum(_ceil(c + n, page) for c, n in zip(context, new)) + spare
    pool = (torch.randperm(need, generator=g) + 7).tolist()
    table = []
    for c in context:
        own = [pool.pop() for _ in range(_ceil(c, page))]
        table.append(own + [-9] * (width - len(own)))
    return pool, table


def _gpu(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check(got, table, want):
    assert table.tolist() == want["table"]
    for name in ("seq_lens", "query_start", "slots", "positions", "requests", "cursor"):
        assert getattr(got, name).tolist() == want[name], name
    assert got.slots.dtype == torch.int64


def _ragged(batch, top, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, top + 1, (batch,), generator=g).tolist()


@pytest.mark.parametrize("page", [1, 16, 24, 64])
@pytest.mark.parametrize("context,new,pad", [
    ([0], [1], 0), ([5], [0], 3), ([0], [0], 0), ([15, 16, 17, 0], [1, 1, 1, 1], 4),
    ([0, 0, 0], [33, 0, 257], 1), (_ragged(37, 300, 1), _ragged(37, 3, 2), 5),
    (_ragged(513, 90, 3), _ragged(513, 40, 4), 0), (_ragged(2049, 20, 5), [1] * 2049, 15)])
def test_matches_the_loop(page, context, new, pad):
    width = max(_ceil(c + n, page) for c, n in zip(context, new)) + 2
    free, table = _inputs(context, new, page, width)
    tokens = sum(new) + pad
    want = _reference(context, new, free, table, page, tokens)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    t = _gpu(table)
    args = (_gpu(context), _gpu(new), _gpu(free), t, page, tokens)
    got = dg.build_block_tables(*args, status=status)
    _check(got, t, want)
    # Repeated, into the same tensors: it reads nothing that it writes.
    again = dg.build_block_tables(*args, out=got, status=status)
    assert again is got
    _check(got, t, want)
    assert int(status) == 0


def test_table_rows_inside_a_wider_tensor_and_a_cursor():
    context, new, page = [40, 0, 7], [30, 50, 1], 16
    free, table = _inputs(context, new, page, 6)
    whole = torch.full((3, 11), -5, dtype=torch.int32, device="cuda")
    view = whole[:, 2:8]
    view.copy_(_gpu(table))
    free = [99, 98] + free
    want = _reference(context, new, free, table, page, 90, cursor=2)
    got = dg.build_block_tables(_gpu(context), _gpu(new), _gpu(free), view, page, 90, cursor=_gpu([2]))
    _check(got, view, want)
    assert (whole[:, :2] == -5).all() and (whole[:, 8:] == -5).all()


def test_steps_follow_one_another_on_a_stream_in_a_graph():
    """Three decode steps from one captured graph: lengths and cursor go round."""
    batch, page, width = 33, 8, 20
    context = _ragged(batch, 60, 8)
    free, table = _inputs(context, [40] * batch, page, width)
    lens, cursor, t, f = _gpu(context), _gpu([0]), _gpu(table), _gpu(free)
    new = torch.ones(batch, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dg.build_block_tables(lens, new, f, t.clone(), page, 40)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = dg.build_block_tables(lens, new, f, t, page, 40, cursor=cursor)
            lens.copy_(got.seq_lens)
            cursor.copy_(got.cursor)
        at = 0
        for _ in range(3):
            graph.replay()
            want = _reference(context, [1] * batch, free, table, page, 40, cursor=at)
            side.synchronize()
            _check(got, t, want)
            context, table, at = want["seq_lens"], want["table"], want["cursor"][0]


def test_what_only_the_gpu_can_see_is_reported():
    def run(context, new, free, width, tokens, page=4):
        t = torch.full((len(context), width), -9, dtype=torch.int32, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        guard = torch.full((tokens + 64,), -77, dtype=torch.int64, device="cuda")
        got = dg.build_block_tables(_gpu(context), _gpu(new), _gpu(free), t, page, tokens, status=status)
        del guard
        return got, t.tolist(), int(status)
    # Pool: 2 pages for 3; the third page and its tokens stay at -1.
    got, t, code = run([0, 0], [8, 4], [5, 6], 4, 12)
    assert code == _lib.ERR_POOL and t == [[5, 6, -9, -9], [-1, -9, -9, -9]]
    assert got.slots.tolist() == [20, 21, 22, 23, 24, 25, 26, 27, -1, -1, -1, -1] and got.cursor.tolist() == [2]
    # Table rows of 1 page.
    got, t, code = run([0, 2], [6, 2], [5, 6, 7], 1, 8)
    assert code == _lib.ERR_TABLE_WIDTH and t[0] == [5]
    assert got.slots.tolist()[:6] == [20, 21, 22, 23, -1, -1] and got.seq_lens.tolist() == [6, 4]
    # More tokens than room.
    got, t, code = run([0], [9], [1, 2, 3], 4, 5)
    assert code == _lib.ERR_TOKENS and got.slots.tolist() == [4, 5, 6, 7, 8] and got.query_start.tolist() == [0, 9]
    # Lengths below zero count as zero; sums past an int are held there.
    got, t, code = run([-3, 0], [2, -5], [1, 2], 4, 4)
    assert code == _lib.ERR_LENGTH and got.slots.tolist() == [4, 5, -1, -1] and got.seq_lens.tolist() == [2, 0]
    big = 2 ** 31 - 1
    got, t, code = run([5, 0], [big, big], [1, 2], 4, 4)
    assert code != 0 and got.query_start.tolist() == [0, big - 5, big]


def test_refusals():
    c, n, f = _gpu([1, 2]), _gpu([1, 1]), _gpu([3, 4])
    t = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    ok = dict(context_lens=c, new_lens=n, free_pages=f, block_table=t, page_size=4, num_tokens=2)
    for bad in (dict(context_lens=c.long()), dict(context_lens=c.cpu()), dict(new_lens=n[:1]), dict(new_lens=n.cpu()),
                dict(free_pages=f.float()), dict(block_table=t.T), dict(block_table=t.long()), dict(block_table=t[:1]),
                dict(page_size=0), dict(num_tokens=-1), dict(cursor=c), dict(status=c.float()),
                dict(block_table=t[:1].expand(2, 4))):
        with pytest.raises(ValueError):
            dg.build_block_tables(**{**ok, **bad})
    step = dg.build_block_tables(**ok)
    with pytest.raises(ValueError):
        dg.build_block_tables(**{**ok, "num_tokens": 3}, out=step)
