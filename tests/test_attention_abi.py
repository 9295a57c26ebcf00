"""CPU tests of the attention operators' C ABI and host logic (no launches):
struct layouts, refusals, status codes, and the rules by which the attention
kernel cuts its work."""

import ctypes
import os
import shutil
import subprocess

import pytest

import decode_opt_b200 as dg
from decode_opt_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD = dg.CUDA_ERROR_INVALID_VALUE


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_match_header(tmp_path):
    structs = {"dg_block_tables": _lib.DgBlockTables, "dg_rotary_args": _lib.DgRotaryArgs,
               "dg_attention_args": _lib.DgAttentionArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "decode_attention_b200.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'  printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    names = {"DG_TYPE_BF16": _lib.TYPE_BF16, "DG_TYPE_FP16": _lib.TYPE_FP16, "DG_TYPE_FP32": _lib.TYPE_FP32,
             "DG_TYPE_E4M3": _lib.TYPE_E4M3, "DG_PAIR_HALF": _lib.PAIR_HALF, "DG_PAIR_ADJACENT": _lib.PAIR_ADJACENT,
             "DG_MAX_ROT": _lib.MAX_ROT, "DG_ERR_LENGTH": _lib.ERR_LENGTH, "DG_ERR_POOL": _lib.ERR_POOL,
             "DG_ERR_TABLE_WIDTH": _lib.ERR_TABLE_WIDTH, "DG_ERR_TOKENS": _lib.ERR_TOKENS,
             "DG_ERR_POSITION": _lib.ERR_POSITION, "DG_ERR_SLOT": _lib.ERR_SLOT, "DG_ERR_PAGE": _lib.ERR_PAGE,
             "DG_ERR_SEQ_LEN": _lib.ERR_SEQ_LEN}
    lines += [f'  printf("value {n} %d\\n", {n});' for n in names]
    lines += ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
                    str(src), "-o", str(exe)], check=True)
    got = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, val = line.split()
        got[(name, field)] = int(val)
    for cname, py in structs.items():
        assert got[(cname, "size")] == ctypes.sizeof(py), cname
        for fname, _ in py._fields_:
            assert got[(cname, fname)] == getattr(py, fname).offset, (cname, fname)
    for n, v in names.items():
        assert got[("value", n)] == v, n


def test_status_codes_have_words():
    codes = [_lib.ERR_LENGTH, _lib.ERR_POOL, _lib.ERR_TABLE_WIDTH, _lib.ERR_TOKENS, _lib.ERR_POSITION, _lib.ERR_SLOT,
             _lib.ERR_PAGE, _lib.ERR_SEQ_LEN]
    words = [dg.status_string(c) for c in codes]
    assert len(set(words)) == len(words) and "unknown status" not in words


def _tables(**kw):
    a = dict(batch=2, page_size=16, table_width=4, num_tokens=8, free_count=4, table_stride=4, context_lens=16,
             new_lens=32, free_pages=48, cursor_in=None, block_table=64, seq_lens=80, query_start=96, slots=112,
             positions=128, requests=144, cursor_out=160, status=None)
    a.update(kw)
    return _lib.lib().dg_build_block_tables(ctypes.byref(_lib.DgBlockTables(**a)), None, 0)


@pytest.mark.parametrize("kw", [
    dict(batch=0), dict(batch=16385), dict(page_size=0), dict(table_width=0), dict(num_tokens=-1), dict(free_count=-1),
    dict(table_stride=3), dict(context_lens=None), dict(new_lens=None), dict(free_pages=None), dict(block_table=None),
    dict(seq_lens=None), dict(query_start=None), dict(cursor_out=None), dict(slots=None), dict(positions=None),
    dict(requests=None), dict(slots=116), dict(seq_lens=16), dict(seq_lens=32),
    dict(cursor_in=160)])
def test_block_tables_refusals(kw):
    assert _tables(**kw) == BAD


def _rotary(**kw):
    a = dict(tokens=4, heads=2, kv_heads=2, head_dim=64, rot=64, type=_lib.TYPE_BF16, cache_type=_lib.TYPE_BF16,
             pairing=0, inverse=0, position_64=1, max_position=100, page_size=16, num_pages=4, q=256, k=512, v=768,
             q_out=1024, k_out=None, k_cache=2048, v_cache=4096, q_stride=(128, 64), k_stride=(128, 64),
             v_stride=(128, 64), q_out_stride=(128, 64), k_out_stride=(0, 0), k_cache_stride=(2048, 128, 64),
             v_cache_stride=(2048, 128, 64), positions=16, position_stride=0, slots=32, cos_sin=64, k_scale=None,
             v_scale=None, status=None)
    a.update(kw)
    return _lib.lib().dg_rotary(ctypes.byref(_lib.DgRotaryArgs(**a)), None, 0)


@pytest.mark.parametrize("kw", [
    dict(tokens=0), dict(head_dim=1), dict(head_dim=2050), dict(rot=0), dict(rot=3), dict(rot=66), dict(head_dim=1024, rot=514),
    dict(max_position=0), dict(type=_lib.TYPE_E4M3), dict(type=_lib.TYPE_FP32), dict(type=7), dict(pairing=2),
    dict(positions=None), dict(cos_sin=None), dict(position_stride=-1), dict(q=None), dict(q_out=None), dict(heads=0),
    dict(k=None), dict(v=None), dict(k_cache=None), dict(v_cache=None), dict(slots=None), dict(page_size=0),
    dict(num_pages=0), dict(cache_type=_lib.TYPE_FP16), dict(k_scale=16), dict(v_scale=16), dict(heads=-1),
    dict(k_cache=None, v_cache=None, v=None), dict(q_stride=(1 << 30, 64)), dict(v_stride=(-128, 64))])
def test_rotary_refusals(kw):
    assert _rotary(**kw) == BAD


def _attention(**kw):
    need = _lib.lib().dg_attention_workspace_bytes()
    a = dict(batch=2, heads=8, kv_heads=2, head_dim=128, page_size=16, num_pages=4, table_width=4,
             type=_lib.TYPE_BF16, cache_type=_lib.TYPE_BF16, window=0, scale=1.0, softcap=0.0, q=256, k_cache=512,
             v_cache=1024, q_stride=(1024, 128), k_cache_stride=(4096, 256, 128), v_cache_stride=(4096, 256, 128),
             block_table=16, table_stride=4, seq_lens=32, k_scale=None, v_scale=None, out=2048, out_stride=(1024, 128),
             lse=None, q_out=None, q_scales=None, workspace=4096, workspace_bytes=need, status=None)
    a.update(kw)
    return _lib.lib().dg_paged_attention(ctypes.byref(_lib.DgAttentionArgs(**a)), None, 0)


@pytest.mark.parametrize("kw", [
    dict(batch=0), dict(heads=0), dict(kv_heads=0), dict(heads=7), dict(head_dim=0), dict(head_dim=4),
    dict(head_dim=12), dict(head_dim=264), dict(page_size=0), dict(num_pages=0), dict(table_width=0),
    dict(table_stride=3), dict(type=_lib.TYPE_FP32, cache_type=_lib.TYPE_FP32), dict(type=_lib.TYPE_E4M3),
    dict(cache_type=_lib.TYPE_FP16), dict(cache_type=9), dict(cache_type=_lib.TYPE_E4M3, head_dim=24),
    dict(window=-1), dict(softcap=-1.0), dict(softcap=float("nan")), dict(scale=float("nan")), dict(q=None),
    dict(k_cache=None), dict(v_cache=None), dict(block_table=None), dict(seq_lens=None), dict(out=None),
    dict(workspace=None), dict(workspace=4104), dict(workspace_bytes=0), dict(q=258), dict(q_stride=(1025, 128)),
    dict(q_stride=(1024, 127)), dict(k_cache=520), dict(v_cache=1032), dict(k_cache_stride=(4097, 256, 128)),
    dict(v_cache_stride=(4096, 257, 128)), dict(v_cache_stride=(4096, 256, 132)), dict(k_scale=16), dict(v_scale=16),
    dict(q_out=16), dict(q_scales=16), dict(q_out=16, q_scales=32, head_dim=64),
    dict(q_out=16, q_scales=32, type=_lib.TYPE_FP16, cache_type=_lib.TYPE_FP16)])
def test_attention_refusals(kw):
    assert _attention(**kw) == BAD


def test_null_arguments_are_refused():
    L = _lib.lib()
    assert L.dg_build_block_tables(None, None, 0) == BAD
    assert L.dg_rotary(None, None, 0) == BAD
    assert L.dg_paged_attention(None, None, 0) == BAD


def _cut(lens, items, tok, window, ctas, warps, extra=14, extra_solo=1, min_run=8):
    """The attention kernel's cut of a batch: (units, CTAs in use, per CTA its
    shares (request, item, first tile, tiles, unit of the item's first tile,
    the item's tiles, one warp's work or not))."""
    line = []
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        tiles = (n - 1) // tok + 1 - lo // tok if n else 0
        line += [(b, i, tiles, extra_solo if tiles <= warps else extra) for i in range(items)] if tiles else []
    total = sum(t + e for _, _, t, e in line)
    used = min(ctas, -(-total // min_run))
    bounds = [total * c // used for c in range(used + 1)]
    shares, at = [[] for _ in range(used)], 0
    for b, i, tiles, e in line:
        for c in range(used):
            lo, hi = max(bounds[c], at), min(bounds[c + 1], at + tiles + e)
            t0, t1 = max(0, lo - at - e), max(0, min(tiles, hi - at - e))
            if lo < hi and t0 < t1:
                solo = tiles <= warps and t1 - t0 == tiles and bounds[c + 1] - bounds[c] >= 2 * (tiles + e)
                shares[c].append((b, i, t0, t1 - t0, at + e, tiles, solo))
        at += tiles + e
    return total, used, shares


@pytest.mark.parametrize("lens,items,window", [
    ([1], 1, 0), ([2049], 8, 0), ([0, 5, 0, 300, 0], 2, 0), ([17] * 40, 4, 0), ([8191, 1, 33, 0, 4096], 8, 100),
    ([131072], 1, 0), ([1] * 700, 3, 0), ([1000, 0, 64, 65] * 9, 5, 64), ([16] * 3 + [129, 3000], 1, 0)])
@pytest.mark.parametrize("tok,warps", [(16, 8), (32, 8), (16, 4)])
def test_attention_shares_meet(lens, items, window, tok, warps):
    """Every tile belongs to one CTA; the CTAs of a shared item are the run
    c0 .. c1 that its first and last tile name, its shares lie in distinct
    workspace slots (2c, or 2c + 1 for the share that begins the item), and no
    two shared items have the same ticket c0."""
    total, used, shares = _cut(lens, items, tok, window, 148, warps)
    owners, slots, tiles_of = {}, set(), {}
    for c, mine in enumerate(shares):
        assert all(s[2] == 0 for s in mine[1:])
        for b, i, t0, count, first, tiles, solo in mine:
            c0 = ((first + 1) * used - 1) // total
            c1 = ((first + tiles) * used - 1) // total
            assert c0 <= c <= c1 and not (solo and c0 != c1)
            owners.setdefault((b, i), []).append((c, c0, c1, t0, count))
            tiles_of[b, i] = tiles
            if count < tiles:
                slot = 2 * c + (1 if t0 == 0 else 0)
                assert slot not in slots and slot == 2 * c + (1 if c == c0 else 0)
                slots.add(slot)
    live = [n for n in lens if n]
    assert len(owners) == len(live) * items
    tickets = set()
    for key, runs in owners.items():
        c0, c1 = runs[0][1:3]
        assert [r[0] for r in runs] == list(range(c0, c1 + 1))
        at = 0
        for _, _, _, t0, count in runs:
            assert t0 == at
            at += count
        assert at == tiles_of[key]
        if c1 > c0:
            assert c0 not in tickets
            tickets.add(c0)


@pytest.mark.parametrize("rows,wide", [(32, 8), (16, 16)])
def test_attention_stage_swizzle_is_free_of_conflicts(rows, wide):
    """The stage layouts of the attention kernel: a permutation of each row's
    16-byte chunks under which the chunks of one load phase fall into 8
    different bank groups (chunk index mod 8)."""
    def e4m3(r, c):
        return c ^ ((r & 6) ^ ((r & 1) << 2))

    def sixteen(r, c):
        return c ^ (r & 7)
    for f in (e4m3, sixteen):
        for r in range(rows):
            assert sorted(f(r, c) for c in range(wide)) == list(range(wide))
    for r in range(0, rows, 8):
        for c in range(wide):
            assert len({sixteen(r + i, c) % 8 for i in range(8)}) == 8
    for r in range(0, rows, 2):
        for c in range(0, wide, 4):
            assert len({e4m3(r + i, c + j) % 8 for i in range(2) for j in range(4)}) == 8
    for r in (0, 1, 8, 9):
        for c in range(0, wide, 2):
            assert len({e4m3(r + 2 * i, c + j) % 8 for i in range(4) for j in range(2)}) == 8
