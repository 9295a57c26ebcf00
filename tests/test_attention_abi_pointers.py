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


def _rotary(**kw):
    a = dict(tokens=4, heads=2, kv_heads=2, head_dim=64, rot=64, type=_lib.TYPE_BF16, cache_type=_lib.TYPE_BF16,
             position_64=1, max_position=100, page_size=16, num_pages=4, q=0x100, k=0x200, v=0x300, q_out=0x400,
             k_cache=0x1000, v_cache=0x2000, q_stride=(128, 64), k_stride=(128, 64), v_stride=(128, 64),
             q_out_stride=(128, 64), k_out_stride=(128, 64), k_cache_stride=(2048, 128, 64),
             v_cache_stride=(2048, 128, 64), positions=0x500, slots=0x600, cos_sin=0x700)
    a.update(kw)
    return _lib.lib().dg_rotary(ctypes.byref(_lib.DgRotaryArgs(**a)), None, 0)


def _attention(**kw):
    need = _lib.lib().dg_attention_workspace_bytes()
    a = dict(batch=2, heads=8, kv_heads=2, head_dim=128, page_size=16, num_pages=4, table_width=4,
             type=_lib.TYPE_BF16, cache_type=_lib.TYPE_BF16, scale=1.0, q=0x100, k_cache=0x1000, v_cache=0x2000,
             q_stride=(1024, 128), k_cache_stride=(4096, 256, 128), v_cache_stride=(4096, 256, 128), block_table=0x200,
             table_stride=4, seq_lens=0x300, out=0x400, out_stride=(1024, 128), workspace=0x4000, workspace_bytes=need)
    a.update(kw)
    return _lib.lib().dg_paged_attention(ctypes.byref(_lib.DgAttentionArgs(**a)), None, 0)


E4M3 = dict(cache_type=_lib.TYPE_E4M3)
FP32 = dict(type=_lib.TYPE_FP32, cache_type=_lib.TYPE_FP32, v=None, k_cache=None, v_cache=None, slots=None, k_out=0x800)


@pytest.mark.parametrize("call,fields,by,kw", [
    (_tables, ("context_lens", "new_lens", "free_pages", "cursor_in", "block_table", "seq_lens", "query_start",
               "positions", "requests", "cursor_out", "status"), (1, 2, 3), {}),
    (_tables, ("slots",), (1, 2, 4), {}),
    (_rotary, ("q", "k", "v", "q_out", "k_out", "k_cache", "v_cache"), (1,), {}),
    (_rotary, ("q", "k", "q_out", "k_out"), (1, 2, 3), FP32),
    (_rotary, ("cos_sin", "status"), (1, 2), {}),
    (_rotary, ("k_scale", "v_scale"), (1, 2), E4M3),
    (_rotary, ("positions", "slots"), (1, 4), {}),
    (_rotary, ("positions",), (1, 2), dict(position_64=0)),
    (_attention, ("out",), (1,), {}),
    (_attention, ("block_table", "seq_lens", "lse", "status"), (1, 2), {}),
    (_attention, ("k_scale", "v_scale"), (1, 2), E4M3),
    (_attention, ("q_scales",), (1, 2), dict(q_out=0x900))])
def test_addresses_between_elements_are_refused(call, fields, by, kw):
    """The GPU would fault on them.  (Whole ones go on to the launch, which a
    host without a GPU answers with another error.)"""
    for name in fields:
        for off in by:
            assert call(**{**kw, name: 0x10000 + off}) == BAD, (name, off)
