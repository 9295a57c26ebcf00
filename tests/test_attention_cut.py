"""CPU test of the walk by which the attention kernel's CTAs go through their
shares of the line of tiles, with the constants and the whole numbers of the
kernel (read from its source), for its three warp counts: every tile is taken
once, by one warp, shares of an item meet in distinct workspace slots under one
ticket, and all of the item's CTAs agree on their number."""

import os
import random
import re

import pytest

from decode_opt_b200 import build

SOURCE = open(os.path.join(build.CSRC, "dg_attention.cu")).read()


def _constant(pattern):
    (found,) = re.findall(pattern, SOURCE)
    return [int(x) for x in found] if isinstance(found, tuple) else int(found)


SOLO = _constant(r"int SOLO = (\d+);")
EXTRA_SOLO, EXTRA_8, EXTRA_16 = _constant(r"int EXTRA_SOLO = (\d+), EXTRA = ROWS_ == 8 \? (\d+) : (\d+);")
MIN_RUN = _constant(r"int MIN_RUN = (\d+);")
MAX_CTAS = _constant(r"int kMaxCtas = (\d+);")


class Line:
    def __init__(self, lens, items, tok, window, rows, warps):
        self.lens, self.items, self.tok, self.window, self.warps = lens, items, tok, window, warps
        self.most = EXTRA_8 if rows == 8 else EXTRA_16

    def tiles(self, b):
        n = self.lens[b]
        first = max(0, n - self.window) if self.window else 0
        return (n - 1) // self.tok + 1 - first // self.tok if n else 0

    def extra(self, tiles):
        return EXTRA_SOLO if tiles <= SOLO else self.most

    def units(self, b):
        t = self.tiles(b)
        return (t + self.extra(t)) * self.items if t else 0

    def walk(self, cta, used, total):
        """The shares of one CTA: (request, item, x, t0, count, tiles, solo, turn)."""
        x0, x1 = total * cta // used, total * (cta + 1) // used
        base, b = 0, 0
        while x0 >= base + self.units(b):
            base += self.units(b)
            b += 1
        run, turn = x1 - x0, 0
        tiles = self.tiles(b)
        unit = tiles + self.extra(tiles)
        item, into = divmod(x0 - base, unit)
        x, t0 = -into, max(0, into - self.extra(tiles))
        while True:
            e = self.extra(tiles)
            count = min(tiles, run - x - e) - t0
            solo = tiles <= SOLO and count == tiles and run >= 2 * (tiles + e)
            if count <= 0:
                return
            yield b, item, x, t0, count, tiles, solo, turn
            x += tiles + e
            if x >= run:
                return
            turn += solo
            item += 1
            if item == self.items:
                item = 0
                b += 1
                while not self.tiles(b):
                    b += 1
                tiles = self.tiles(b)
            t0 = 0

    def check(self, ctas):
        total = sum(self.units(b) for b in range(len(self.lens)))
        used = min(ctas, -(-total // MIN_RUN))
        taken, slots, tickets, parts = {}, set(), {}, {}
        for c in range(used):
            for b, item, x, t0, count, tiles, solo, turn in self.walk(c, used, total):
                # Tile t of the share is warp t % warps', or all are one warp's.
                for t in range(t0, t0 + count):
                    assert taken.setdefault((b, item, t), c) == c
                assert len({turn % self.warps} if solo else {0}) == 1
                if count == tiles:
                    continue
                assert not solo
                slot = 2 * c + (t0 == 0)
                assert slot not in slots and slot < 2 * MAX_CTAS
                slots.add(slot)
                first = total * c // used + x + self.extra(tiles)
                c0 = ((first + 1) * used - 1) // total
                c1 = ((first + tiles) * used - 1) // total
                assert c0 <= c <= c1 < used and (t0 == 0) == (c == c0)
                assert tickets.setdefault(c0, (b, item)) == (b, item)
                assert parts.setdefault((b, item), (c0, c1, []))[:2] == (c0, c1)
                parts[b, item][2].append(c)
        for c0, c1, cs in parts.values():
            assert cs == list(range(c0, c1 + 1)) and len(cs) <= MAX_CTAS
        want = sum(self.tiles(b) for b in range(len(self.lens))) * self.items
        assert len(taken) == want


@pytest.mark.parametrize("tok,warps", [(32, 12), (16, 8), (32, 8), (16, 4)])
@pytest.mark.parametrize("rows", [8, 16])
@pytest.mark.parametrize("lens,items,window", [
    ([1], 1, 0), ([2049], 8, 0), ([0, 5, 0, 300, 0], 2, 0), ([17] * 40, 4, 0), ([8191, 1, 33, 0, 4096], 8, 100),
    ([131072], 1, 0), ([1] * 700, 3, 0), ([1000, 0, 64, 65] * 9, 5, 64), ([16] * 3 + [129, 3000], 1, 0),
    ([128, 129, 256, 257] * 20, 3, 0), ([20] * 148, 1, 0), ([0] * 5 + [9] + [0] * 300, 1, 0)])
def test_walks(lens, items, window, tok, warps, rows):
    for ctas in (148, 160, 132, 1):
        Line(lens, items, tok, window, rows, warps).check(ctas)


@pytest.mark.parametrize("seed", range(60))
def test_walks_of_any_batch(seed):
    r = random.Random(seed)
    top = int(10 ** r.uniform(0, 4.3))
    lens = [0 if r.random() < 0.1 else r.randint(1, top) for _ in range(int(10 ** r.uniform(0, 2.3)))]
    window = r.choice((0, 0, r.randint(1, top)))
    tok, warps = r.choice(((32, 12), (16, 8), (32, 8), (16, 4)))
    Line(lens, r.randint(1, 12), tok, window, r.choice((8, 16)), warps).check(r.choice((148, 148, r.randint(1, 160))))
