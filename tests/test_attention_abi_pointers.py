"""CPU tests of refused pointers of the attention operators' C ABI: nothing is
launched, and no pointer is read."""

import ctypes

import pytest

import decode_opt_b200 as dg
from decode_opt_b200 import _lib

BAD = dg.CUDA_ERROR_INVALID_VALUE


def _tables(**kw):
    a = dict(batch=3, page_size=16, table_width=4, num_tokens=8, free_count=4, table_stride=6, context_lens=0x100,
             new_lens=0x200, free_pages=0x300, block_table=0x1000, seq_lens=0x400, query_start=0x500, slots=0x600,
             positions=0x700, requests=0x800, cursor_out=0x900)
    a.update(kw)
    return _lib.lib().dg_build_block_tables(ctypes.byref(_lib.DgBlockTables(**a)), None, 0)


def _meets(free, count, batch, width, stride, table=0x1000):
    return any(free < table + (b * stride + width) * 4 and table + b * stride * 4 < free + 4 * count
               for b in range(batch))


def test_a_free_list_in_the_table_is_refused():
    """The table's rows are 4 entries of every 6; a list in the gaps or beside
    the table is none of them (and goes on to a launch, which a host without a
    GPU answers otherwise)."""
    met = 0
    for free in range(0x1000 - 48, 0x1000 + 3 * 24 + 48, 4):
        for count in (1, 2, 3, 7, 30):
            if _meets(free, count, 3, 4, 6):
                assert _tables(free_pages=free, free_count=count) == BAD, (hex(free), count)
                met += 1
    assert met > 50


def test_the_rule_is_exact():
    """The rule that finds the one row that can meet the list, against all rows."""
    def rule(free, count, batch, width, stride, table=0x1000):
        row, step = 4 * width, 4 * stride
        b = 0 if free < table + row else (free - table - row) // step + 1
        return count > 0 and b < batch and table + b * step < free + 4 * count
    for batch in (1, 2, 5):
        for width, stride in ((1, 1), (4, 4), (4, 6), (3, 11)):
            for free in range(0x1000 - 60, 0x1000 + 4 * stride * batch + 60, 4):
                for count in (0, 1, 2, 5, 13, 100):
                    want = count > 0 and _meets(free, count, batch, width, stride)
                    assert rule(free, count, batch, width, stride) == want
