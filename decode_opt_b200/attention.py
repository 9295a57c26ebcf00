"""The operators between a decode layer's products: block tables and slot maps
from request lengths, rotary positions with several axes, the write into a
paged key-value cache, and the attention of one new token over it
(include/decode_attention_b200.h; no counterpart in the reference).

One serving step::

    step = dg.build_block_tables(context_lens, new_lens, free_pages, block_table, page_size, num_tokens)
    for layer in layers:
        q = dg.rotary_append(q, k, v, step.positions, step.slots, k_cache, v_cache, table)
        out = dg.paged_attention(q, k_cache, v_cache, block_table, step.seq_lens)

Tensors are CUDA tensors whose last dimension is contiguous; other strides are
free (a fused projection's slices, a cache kept head by head), within the
alignments that each function names.  Arguments that cannot be served raise
ValueError before anything is launched.  What only the GPU can see (lengths,
pages, slots, positions) is checked there: the access is left out and `status`,
an optional zeroed int32 tensor, receives a code (:func:`status_string`).
Nothing synchronises; every call can be captured in a CUDA graph.  `stream`
(default: the current one) takes a torch stream or a cudaStream_t handle;
outputs made here are allocated on it.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import struct
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

__all__ = ["StepTables", "build_block_tables", "rope_table", "rotary", "rotary_append", "paged_attention",
           "attention_workspace"]

_TYPE = {torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_FP16, torch.float32: _lib.TYPE_FP32}
_CACHE_TYPE = {torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_FP16,
               torch.float8_e4m3fn: _lib.TYPE_E4M3, torch.uint8: _lib.TYPE_E4M3}
_PAIRING = {"half": _lib.PAIR_HALF, "adjacent": _lib.PAIR_ADJACENT}
_INT32_MAX = 2 ** 31 - 1


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _addr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _layout(struct_type) -> struct.Struct:
    """A ctypes mirror as a struct.Struct of its members in order (arrays
    spread out): packing one is ten times cheaper than filling the mirror, and
    the calls of a decode step are short."""
    code = {ctypes.c_int: "i", ctypes.c_uint: "I", ctypes.c_float: "f", ctypes.c_longlong: "q",
            ctypes.c_ulonglong: "Q", ctypes.c_void_p: "P"}
    form = "@"
    for _, t in struct_type._fields_:
        form += code[t] if t in code else f"{t._length_}{code[t._type_]}"
    layout = struct.Struct(form)
    assert layout.size <= ctypes.sizeof(struct_type) < layout.size + 8
    # Trailing padding, so that the bytes are a whole C struct.
    return struct.Struct(form + f"{ctypes.sizeof(struct_type) - layout.size}x")


_PACK_TABLES = _layout(_lib.DgBlockTables).pack
_PACK_ROTARY = _layout(_lib.DgRotaryArgs).pack
_PACK_ATTENTION = _layout(_lib.DgAttentionArgs).pack


@contextlib.contextmanager
def _on(device, stream):
    """With `device` current and, where one is given, `stream` too."""
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            s = torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream
            with torch.cuda.stream(s):
                yield


def _elsewhere(device, stream) -> bool:
    """Whether the call has to be made under :func:`_on` first."""
    return stream is not None or torch.cuda.current_device() != device.index


def _launch(name: str, args: bytes, device, pdl_attr) -> None:
    rc = getattr(_lib.lib(), name)(args, torch._C._cuda_getCurrentRawStream(device.index), 1 if pdl_attr else 0)
    if rc != 0:
        raise RuntimeError(f"{name} failed: cudaError {rc}")


def _check_ints(name: str, t, count: int, device, dtype=torch.int32) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != count or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {count} values on {device}")


def _check_status(status, device) -> None:
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1 or status.device != device):
        raise ValueError(f"status must be an int32 tensor on {device}")


def _check_block_table(t, batch: int, device) -> Tuple[int, int]:
    """(entries a row, row stride) of a block table."""
    if t.dtype != torch.int32 or t.dim() != 2 or t.device != device:
        raise ValueError(f"block_table must be int32 [{batch}, width] on {device}")
    rows, width = t.shape
    stride, unit = t.stride()
    if rows != batch or width < 1 or (unit != 1 and width > 1) or (stride < width and batch > 1):
        raise ValueError(f"block_table must be [{batch}, width >= 1] with unit column stride and rows that do not overlap")
    return width, stride if batch > 1 else width


# ---------------------------------------------------------------------------
# Block tables and slot maps
# ---------------------------------------------------------------------------

@dataclass
class StepTables:
    """What :func:`build_block_tables` makes for one step (all on the GPU)."""

    seq_lens: torch.Tensor      # [B] int32: tokens of each request after the step
    query_start: torch.Tensor   # [B + 1] int32: each request's first new token, and their number
    slots: torch.Tensor         # [num_tokens] int64: page * page_size + offset; -1 for padding
    positions: torch.Tensor     # [num_tokens] int32: position in the request; 0 for padding
    requests: torch.Tensor      # [num_tokens] int32: the token's request; -1 for padding
    cursor: torch.Tensor        # [1] int32: the next page of the free list


def build_block_tables(context_lens, new_lens, free_pages, block_table, page_size: int, num_tokens: int, *,
                       cursor=None, out: Optional[StepTables] = None, status=None, stream=None,
                       pdl_attr: bool = False) -> StepTables:
    """The paged cache's bookkeeping of one step (``dg_build_block_tables``).

    Request b has ``context_lens[b]`` tokens in the cache and brings
    ``new_lens[b]`` (int32 [B], B <= 16384; zeros are fine).  The pages that it
    lacks are taken, in request order, from ``free_pages[cursor:]`` (int32;
    `cursor` an int32 [1] tensor, default 0) and entered into its row of
    ``block_table`` (int32 [B, W], changed in place; entries that no new page
    needs are left alone).  ``num_tokens`` >= the new tokens' number sizes the
    per-token outputs; the rest is padding, so that a CUDA graph can be
    replayed for any smaller step.  `out` (a previous result of the same sizes)
    is written instead of new tensors."""
    _need(context_lens.is_cuda, "context_lens must be a CUDA tensor")
    device = context_lens.device
    if _elsewhere(device, stream):
        with _on(device, stream):
            return build_block_tables(context_lens, new_lens, free_pages, block_table, page_size, num_tokens,
                                      cursor=cursor, out=out, status=status, pdl_attr=pdl_attr)
    batch, free_count = context_lens.shape[0], free_pages.shape[0]
    _need(1 <= batch <= 16384, "batch must be 1 .. 16384")
    _check_ints("context_lens", context_lens, batch, device)
    _check_ints("new_lens", new_lens, batch, device)
    _check_ints("free_pages", free_pages, free_count, device)
    width, table_stride = _check_block_table(block_table, batch, device)
    _need(1 <= page_size <= _INT32_MAX and 0 <= num_tokens <= _INT32_MAX, "page_size >= 1 and num_tokens >= 0")
    if cursor is not None:
        _check_ints("cursor", cursor, 1, device)
    _check_status(status, device)
    if out is None:
        # One allocation: 8-byte slots, then the 4-byte parts, each begun on 16 bytes.
        tokens, rows, starts = (num_tokens + 3) & ~3, (batch + 3) & ~3, (batch + 4) & ~3
        part = torch.empty(4 * tokens + rows + starts + 4, dtype=torch.int32, device=device)
        slots, positions, requests, seq_lens, query_start, next_page = part.split_with_sizes(
            (2 * tokens, tokens, tokens, rows, starts, 4))
        slots = slots.view(torch.int64)
        if tokens != num_tokens:
            slots, positions, requests = slots[:num_tokens], positions[:num_tokens], requests[:num_tokens]
        out = StepTables(seq_lens if rows == batch else seq_lens[:batch], query_start[:batch + 1], slots, positions,
                         requests, next_page[:1])
    else:
        _check_ints("out.seq_lens", out.seq_lens, batch, device)
        _check_ints("out.query_start", out.query_start, batch + 1, device)
        _check_ints("out.slots", out.slots, num_tokens, device, torch.int64)
        _check_ints("out.positions", out.positions, num_tokens, device)
        _check_ints("out.requests", out.requests, num_tokens, device)
        _check_ints("out.cursor", out.cursor, 1, device)
    args = _PACK_TABLES(batch, page_size, width, num_tokens, free_count, table_stride, context_lens.data_ptr(),
                        new_lens.data_ptr(), free_pages.data_ptr(), _addr(cursor), block_table.data_ptr(),
                        out.seq_lens.data_ptr(), out.query_start.data_ptr(), out.slots.data_ptr(),
                        out.positions.data_ptr(), out.requests.data_ptr(), out.cursor.data_ptr(), _addr(status))
    _launch("dg_build_block_tables", args, device, pdl_attr)
    return out


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------

def rope_table(max_position: int, rot: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos | sin of ``p * theta ** (-2i / rot)``, fp32 [max_position, rot]: made
    once, in 64 bits, for :func:`rotary` and :func:`rotary_append`."""
    _need(max_position >= 1 and rot >= 2 and rot % 2 == 0, "max_position >= 1 and an even rot >= 2")
    freq = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


@functools.lru_cache(maxsize=64)
def _axis_words(sections: Optional[Tuple[int, ...]], interleaved: bool, half: int):
    """(axes, the packed axis of each pair) of `sections`."""
    if sections is None:
        sections = (half,)
    if not 1 <= len(sections) <= 4 or any(s < 0 for s in sections) or sum(sections) != half:
        raise ValueError(f"sections must be 1 to 4 counts that add up to rot / 2 = {half}, got {sections}")
    if interleaved:
        left, axes = list(sections), []
        while len(axes) < half:
            for a in range(len(left)):
                if left[a]:
                    left[a] -= 1
                    axes.append(a)
    else:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    words = [0] * (_lib.MAX_ROT // 32)
    for i, a in enumerate(axes):
        words[i // 16] |= a << (2 * (i % 16))
    return len(sections), tuple(words)


def _heads_of(name: str, t, tokens: int, dim: int, dtype, device):
    """(heads, (token stride, head stride)) of a [tokens, heads, dim] tensor."""
    if t.dim() != 3 or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} [{tokens}, heads, {dim}] on {device}")
    n, heads, d = t.shape
    s0, s1, unit = t.stride()
    if n != tokens or d != dim or heads < 1 or unit != 1 or max(s0, s1) > 0x1fffffff:
        raise ValueError(f"{name} must be [{tokens}, heads >= 1, {dim}] with unit last stride and strides below 2^29")
    return heads, (s0, s1)


def _cache_of(k_cache, v_cache, heads: int, dim: int, dtype, device):
    """(type, pages, page size, strides of k_cache, strides of v_cache)."""
    kind = k_cache.dtype
    code = _CACHE_TYPE.get(kind)
    if code is None or (code != _lib.TYPE_E4M3 and kind != dtype) or v_cache.dtype != kind:
        raise ValueError(f"both caches must be {dtype} or e4m3 (float8_e4m3fn or uint8), got {kind}, {v_cache.dtype}")
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or k_cache.device != device or v_cache.device != device:
        raise ValueError(f"both caches must be [pages, page_size, {heads}, {dim}] on {device}")
    pages, page_size, h, d = shape
    if h != heads or d != dim or ks[3] != 1 or vs[3] != 1 or not 1 <= pages <= _INT32_MAX or page_size < 1:
        raise ValueError(f"the caches must be [pages >= 1, page_size >= 1, {heads}, {dim}] with unit last stride")
    return code, pages, page_size, ks[:3], vs[:3]


def _check_scale(name: str, t, heads: int, code: int, device) -> None:
    if code != _lib.TYPE_E4M3:
        raise ValueError(f"{name} goes with an e4m3 cache")
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != heads or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be fp32 [{heads}] on {device}")


_NO2, _NO3 = (0, 0), (0, 0, 0)


def _rotary(q, k, v, positions, table, sections, interleaved, pairing, inverse, q_out, k_out, caches, slots, k_scale,
            v_scale, status, pdl_attr):
    """dg_rotary on the current device and stream; returns (q_out, k_out), made
    here where they are True."""
    x = q if q is not None else k
    dtype, device = x.dtype, x.device
    kind = _TYPE.get(dtype)
    _need(kind is not None and x.dim() == 3, "q and k must be bf16, fp16 or fp32 [tokens, heads, dim]")
    tokens, _, dim = x.shape
    _need(tokens >= 1 and 2 <= dim <= 2048, "q and k need at least one token and a dim of 2 .. 2048")
    heads = kv_heads = code = pages = page_size = 0
    qs = ks = vs = qos = kos = _NO2
    kcs = vcs = _NO3
    if q is not None:
        heads, qs = _heads_of("q", q, tokens, dim, dtype, device)
    if k is not None:
        kv_heads, ks = _heads_of("k", k, tokens, dim, dtype, device)
    if table.dtype != torch.float32 or table.dim() != 2 or table.device != device or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous fp32 [max_position, rot] tensor on {device}")
    max_position, rot = table.shape
    if max_position < 1 or rot < 2 or rot % 2 != 0 or rot > dim or rot > _lib.MAX_ROT:
        raise ValueError(f"the table's width must be even and at most {min(dim, _lib.MAX_ROT)}")
    _need(pairing in _PAIRING, "pairing must be 'half' or 'adjacent'")
    axes, words = _axis_words(None if sections is None else tuple(sections), bool(interleaved), rot // 2)
    wide = positions.dtype == torch.int64
    shape, strides = positions.shape, positions.stride()
    if not (wide or positions.dtype == torch.int32) or positions.device != device or len(shape) not in (1, 2) or \
            shape[-1] != tokens or (strides[-1] != 1 and tokens > 1):
        raise ValueError(f"positions must be int32 or int64 [{tokens}] or [axes, {tokens}] on {device}")
    position_stride = 0
    if len(shape) == 2:
        _need(shape[0] == axes, f"positions has {shape[0]} axes, the sections {axes}")
        position_stride = strides[0] if axes > 1 else 0
        _need(position_stride >= 0, "positions must not run backwards")
    if status is not None:
        _check_status(status, device)
    k_cache = v_cache = None
    if caches is not None:
        k_cache, v_cache = caches
        v_heads, vs = _heads_of("v", v, tokens, dim, dtype, device)
        _need(v_heads == kv_heads, "k and v must have one shape")
        _need(dtype != torch.float32, "the cache write takes bf16 or fp16")
        code, pages, page_size, kcs, vcs = _cache_of(k_cache, v_cache, kv_heads, dim, dtype, device)
        _check_ints("slots", slots, tokens, device, torch.int64)
        if k_scale is not None:
            _check_scale("k_scale", k_scale, kv_heads, code, device)
        if v_scale is not None:
            _check_scale("v_scale", v_scale, kv_heads, code, device)
    if q_out is True:
        q_out, qos = torch.empty((tokens, heads, dim), dtype=dtype, device=device), (heads * dim, dim)
    elif q_out is not None:
        _need(q is not None, "out_q without q")
        n, qos = _heads_of("out_q", q_out, tokens, dim, dtype, device)
        _need(n == heads, "out_q must have q's shape")
    if k_out is True:
        k_out, kos = torch.empty((tokens, kv_heads, dim), dtype=dtype, device=device), (kv_heads * dim, dim)
    elif k_out is not None:
        _need(k is not None, "out_k without k")
        n, kos = _heads_of("out_k", k_out, tokens, dim, dtype, device)
        _need(n == kv_heads, "out_k must have k's shape")
    args = _PACK_ROTARY(
        tokens, heads, kv_heads, dim, rot, kind, code if caches is not None else kind, _PAIRING[pairing],
        1 if inverse else 0, 1 if wide else 0, max_position, page_size, pages, _addr(q), _addr(k), _addr(v),
        _addr(q_out), _addr(k_out), _addr(k_cache), _addr(v_cache), *qs, *ks, *vs, *qos, *kos, *kcs, *vcs,
        positions.data_ptr(), position_stride, _addr(slots), table.data_ptr(), _addr(k_scale), _addr(v_scale),
        _addr(status), *words)
    _launch("dg_rotary", args, device, pdl_attr)
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """rotary() where a gradient is wanted: a rotation's gradient is its
    inverse."""

    @staticmethod
    def forward(ctx, q, k, positions, table, kw):
        ctx.save_for_backward(positions, table)
        ctx.kw = kw
        sections, interleaved, pairing, inverse, status, pdl_attr = kw
        return _rotary(q, k, None, positions, table, sections, interleaved, pairing, inverse, q is not None or None,
                       k is not None or None, None, None, None, None, status, pdl_attr)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, table = ctx.saved_tensors
        sections, interleaved, pairing, inverse = ctx.kw[:4]
        dq, dk = (g if g is None or g.stride(-1) == 1 else g.contiguous() for g in (dq, dk))
        gq = gk = None
        if dq is not None or dk is not None:
            gq, gk = _rotary(dq, dk, None, positions, table, sections, interleaved, pairing, not inverse,
                             dq is not None or None, dk is not None or None, None, None, None, None, None, False)
        return gq, gk, None, None, None


def rotary(q, k, positions, table, *, sections: Optional[Sequence[int]] = None, interleaved: bool = False,
           pairing: str = "half", inverse: bool = False, out_q=None, out_k=None, status=None, stream=None,
           pdl_attr: bool = False):
    """Rotary positions on q [T, Hq, D] and k [T, Hk, D] (bf16, fp16 or fp32;
    either may be None): returns the rotated (q, k) (``dg_rotary``).

    The first ``rot = table.shape[1]`` values of a head turn in pairs, (i, i +
    rot/2) or, with ``pairing="adjacent"``, (2i, 2i + 1); the rest passes.
    `positions` (int32 or int64) is [T], or [axes, T] with `sections`: how many
    of the rot/2 pairs follow each axis -- one axis after the other, or dealt in
    turn (``interleaved``) while an axis has pairs left.  ``inverse`` turns
    back, which is also the gradient; the call is differentiable in q and k.
    `out_q`, `out_k` may be q and k themselves."""
    x = q if q is not None else k
    _need(x is not None and x.is_cuda, "q or k must be a CUDA tensor")
    if _elsewhere(x.device, stream):
        with _on(x.device, stream):
            return rotary(q, k, positions, table, sections=sections, interleaved=interleaved, pairing=pairing,
                          inverse=inverse, out_q=out_q, out_k=out_k, status=status, pdl_attr=pdl_attr)
    if torch.is_grad_enabled() and ((q is not None and q.requires_grad) or (k is not None and k.requires_grad)):
        _need(out_q is None and out_k is None, "out_q and out_k do not go with a gradient")
        return _Rotary.apply(q, k, positions, table, (sections, interleaved, pairing, inverse, status, pdl_attr))
    return _rotary(q, k, None, positions, table, sections, interleaved, pairing, inverse,
                   out_q if out_q is not None else (True if q is not None else None),
                   out_k if out_k is not None else (True if k is not None else None),
                   None, None, None, None, status, pdl_attr)


def rotary_append(q, k, v, positions, slots, k_cache, v_cache, table, *, sections: Optional[Sequence[int]] = None,
                  interleaved: bool = False, pairing: str = "half", k_scale=None, v_scale=None, out_q=None,
                  status=None, stream=None, pdl_attr: bool = False):
    """:func:`rotary` on q and k, with the rotated k and v written into the
    paged cache in the same kernel; returns the rotated q.

    ``k_cache`` and ``v_cache`` are [pages, page_size, Hk, D] in q's type (bf16
    or fp16) or e4m3 (float8_e4m3fn or uint8): then ``e4m3(clamp(x /
    scale[head], +-448))`` is stored, `k_scale` and `v_scale` fp32 [Hk] or None
    for 1.  ``slots[t] = page * page_size + offset`` (int64; below 0: the token
    is not cached).  Slots of one call must differ."""
    _need(q is not None and k is not None and v is not None and q.is_cuda, "rotary_append takes CUDA tensors q, k and v")
    if _elsewhere(q.device, stream):
        with _on(q.device, stream):
            return rotary_append(q, k, v, positions, slots, k_cache, v_cache, table, sections=sections,
                                 interleaved=interleaved, pairing=pairing, k_scale=k_scale, v_scale=v_scale,
                                 out_q=out_q, status=status, pdl_attr=pdl_attr)
    return _rotary(q, k, v, positions, table, sections, interleaved, pairing, False,
                   out_q if out_q is not None else True, None, (k_cache, v_cache), slots, k_scale, v_scale, status,
                   pdl_attr)[0]


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

_ATTENTION_WORKSPACES: dict = {}
_TICKET_BYTES = 1024


@functools.lru_cache(maxsize=None)
def _workspace_bytes() -> int:
    return int(_lib.lib().dg_attention_workspace_bytes())


def attention_workspace(device="cuda") -> torch.Tensor:
    """A workspace for :func:`paged_attention` (about 5 MB, any arguments).
    Calls that can overlap on the GPU need one each."""
    ws = torch.empty(_workspace_bytes(), dtype=torch.uint8, device=device)
    ws[:_TICKET_BYTES].zero_()               # the tickets; the rest is written before it is read
    return ws


def _stream_workspace(device) -> torch.Tensor:
    # Kept per stream: calls on one stream run one after another.  A captured
    # graph may be replayed on any stream, so it gets its own, from its pool.
    if torch.cuda.is_current_stream_capturing():
        return attention_workspace(device)
    key = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
    ws = _ATTENTION_WORKSPACES.get(key)
    if ws is None:
        ws = _ATTENTION_WORKSPACES[key] = attention_workspace(device)
    return ws


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, *, scale: Optional[float] = None,
                    window: Optional[int] = None, softcap: Optional[float] = None, k_scale=None, v_scale=None,
                    out=None, return_lse: bool = False, q_out=None, q_scales=None, workspace=None, status=None,
                    stream=None, pdl_attr: bool = False):
    """Attention of one new token per request over its paged cache
    (``dg_paged_attention``): out [B, Hq, D] in q's type, or (out, lse) with
    ``return_lse`` (fp32 [B, Hq], natural logarithm).

    q [B, Hq, D] is bf16 or fp16 (even strides); the caches are [pages,
    page_size, Hk, D] in q's type or e4m3 with optional per-head scales (strides
    and addresses multiples of 16 bytes), Hq a multiple of Hk, D a multiple of
    8 (e4m3: 16) up to 256.  ``seq_lens[b]`` (int32, the new token included)
    tokens of request b are seen, or the last `window` of them; token t lies in
    page ``block_table[b, t // page_size]`` (int32).  No live token: 0, lse
    -inf.  `scale` defaults to D ** -0.5; `softcap` c: c * tanh(s / c).

    `q_out` (uint8 [B, Hq * D]) and `q_scales` (fp32 [B, Hq * D / 128]) also
    receive the result quantised for the next product, the bytes of
    ``quantize_activation`` (bf16 and D a multiple of 128).  `workspace`: from
    :func:`attention_workspace`; by default one is kept per stream, and a call
    under capture gets its own, zeroed in the graph."""
    _need(q.is_cuda and q.dim() == 3, "q must be a CUDA tensor [batch, heads, dim]")
    device, dtype = q.device, q.dtype
    if _elsewhere(device, stream):
        with _on(device, stream):
            return paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale=scale, window=window,
                                   softcap=softcap, k_scale=k_scale, v_scale=v_scale, out=out, return_lse=return_lse,
                                   q_out=q_out, q_scales=q_scales, workspace=workspace, status=status,
                                   pdl_attr=pdl_attr)
    _need(dtype == torch.bfloat16 or dtype == torch.float16, "q must be bf16 or fp16")
    batch, heads, dim = q.shape
    q0, q1, unit = q.stride()
    q_at, k_at, v_at = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    _need(batch >= 1 and unit == 1 and (q_at | 2 * q0 | 2 * q1) % 4 == 0,
          "q must be [batch >= 1, heads, dim], 4-byte aligned, with unit last and otherwise even strides")
    _need(k_cache.dim() == 4, "the caches must be [pages, page_size, kv_heads, dim]")
    kv_heads = k_cache.shape[2]
    _need(kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0, "heads must be a multiple of the cache's heads")
    code, pages, page_size, ks, vs = _cache_of(k_cache, v_cache, kv_heads, dim, dtype, device)
    unit = 16 if code == _lib.TYPE_E4M3 else 8       # 16 bytes
    _need(8 <= dim <= 256 and dim % unit == 0, f"dim must be a multiple of {unit}, at most 256")
    _need((ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) % unit == 0 and (k_at | v_at) % 16 == 0,
          "the caches must be 16-byte aligned, strides multiples of 16 bytes")
    width, table_stride = _check_block_table(block_table, batch, device)
    _check_ints("seq_lens", seq_lens, batch, device)
    if k_scale is not None:
        _check_scale("k_scale", k_scale, kv_heads, code, device)
    if v_scale is not None:
        _check_scale("v_scale", v_scale, kv_heads, code, device)
    _need(window is None or 1 <= window <= _INT32_MAX, "window must be at least 1")
    _need(softcap is None or 0.0 < softcap < float("inf"), "softcap must be positive")
    if status is not None:
        _check_status(status, device)
    if out is not None:
        n, (o0, o1) = _heads_of("out", out, batch, dim, dtype, device)
        _need(n == heads, "out must have q's shape")
    if q_out is not None or q_scales is not None:
        _need(q_out is not None and q_scales is not None, "q_out and q_scales go together")
        _need(dtype == torch.bfloat16 and dim % 128 == 0, "the quantised result takes bf16 and dim a multiple of 128")
        n = heads * dim
        _need(q_out.dtype in (torch.uint8, torch.float8_e4m3fn) and q_out.shape == (batch, n)
              and q_out.is_contiguous() and q_out.device == device, f"q_out must be uint8 [{batch}, {n}], contiguous")
        _need(q_scales.dtype == torch.float32 and q_scales.shape == (batch, n // 128)
              and q_scales.is_contiguous() and q_scales.device == device,
              f"q_scales must be fp32 [{batch}, {n // 128}], contiguous")
    nbytes = _workspace_bytes()
    if workspace is None:
        workspace = _stream_workspace(device)
    else:
        _need(workspace.device == device and workspace.is_contiguous() and workspace.data_ptr() % 16 == 0
              and workspace.numel() * workspace.element_size() >= nbytes,
              f"workspace must come from attention_workspace({str(device)!r})")
    if out is None:
        out, o0, o1 = torch.empty((batch, heads, dim), dtype=dtype, device=device), heads * dim, dim
    lse = torch.empty((batch, heads), dtype=torch.float32, device=device) if return_lse else None
    args = _PACK_ATTENTION(
        batch, heads, kv_heads, dim, page_size, pages, width, _TYPE[dtype], code, window or 0,
        dim ** -0.5 if scale is None else scale, softcap or 0.0, q_at, k_at, v_at, q0, q1, *ks, *vs,
        block_table.data_ptr(), table_stride, seq_lens.data_ptr(), _addr(k_scale), _addr(v_scale), out.data_ptr(), o0,
        o1, _addr(lse), _addr(q_out), _addr(q_scales), workspace.data_ptr(), nbytes, _addr(status))
    _launch("dg_paged_attention", args, device, pdl_attr)
    return (out, lse) if return_lse else out
