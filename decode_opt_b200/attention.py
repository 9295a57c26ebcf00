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


def _addr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


@contextlib.contextmanager
def _on(device, stream):
    """With `device` current and, where one is given, `stream` too; yields the
    stream's handle."""
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream(device).cuda_stream
        else:
            s = torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream
            with torch.cuda.stream(s):
                yield s.cuda_stream


def _launch(name: str, args, handle, pdl_attr) -> None:
    rc = getattr(_lib.lib(), name)(ctypes.byref(args), handle, int(bool(pdl_attr)))
    if rc != 0:
        raise RuntimeError(f"{name} failed: cudaError {rc}")


def _check_same_device(device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not {device}")


def _check_ints(name: str, t, count: int, dtype=torch.int32) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != count or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {count} values")


def _check_status(status) -> None:
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 tensor")


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
    device, batch = context_lens.device, context_lens.shape[0]
    _need(1 <= batch <= 16384, "batch must be 1 .. 16384")
    _check_ints("context_lens", context_lens, batch)
    _check_ints("new_lens", new_lens, batch)
    _check_ints("free_pages", free_pages, free_pages.shape[0])
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch
          and block_table.shape[1] >= 1 and (block_table.stride(1) == 1 or block_table.shape[1] == 1),
          "block_table must be int32 [batch, width], width >= 1, with unit column stride")
    width = block_table.shape[1]
    table_stride = block_table.stride(0) if batch > 1 else width
    _need(table_stride >= width, "block_table's rows overlap")
    _need(1 <= page_size <= _INT32_MAX and 0 <= num_tokens <= _INT32_MAX, "page_size >= 1 and num_tokens >= 0")
    if cursor is not None:
        _check_ints("cursor", cursor, 1)
    _check_status(status)
    _check_same_device(device, new_lens=new_lens, free_pages=free_pages, block_table=block_table, cursor=cursor,
                       status=status)
    with _on(device, stream) as handle:
        if out is None:
            def ints(n, dtype=torch.int32):
                return torch.empty(n, dtype=dtype, device=device)
            out = StepTables(ints(batch), ints(batch + 1), ints(num_tokens, torch.int64), ints(num_tokens),
                             ints(num_tokens), ints(1))
        else:
            _check_ints("out.seq_lens", out.seq_lens, batch)
            _check_ints("out.query_start", out.query_start, batch + 1)
            _check_ints("out.slots", out.slots, num_tokens, torch.int64)
            _check_ints("out.positions", out.positions, num_tokens)
            _check_ints("out.requests", out.requests, num_tokens)
            _check_ints("out.cursor", out.cursor, 1)
            _check_same_device(device, **vars(out))
        args = _lib.DgBlockTables(batch, page_size, width, num_tokens, free_pages.shape[0], table_stride,
                                  context_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(), _addr(cursor),
                                  block_table.data_ptr(), out.seq_lens.data_ptr(), out.query_start.data_ptr(),
                                  out.slots.data_ptr(), out.positions.data_ptr(), out.requests.data_ptr(),
                                  out.cursor.data_ptr(), _addr(status))
        _launch("dg_build_block_tables", args, handle, pdl_attr)
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
    return len(sections), (ctypes.c_uint * len(words))(*words)


def _heads_of(name: str, t, tokens: int, dim: int, dtype, device):
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != dim or t.dtype != dtype or t.device != device or \
            t.stride(2) != 1:
        raise ValueError(f"{name} must be {dtype} [{tokens}, heads, {dim}] on {device} with unit last stride")


def _check_cache(k_cache, v_cache, heads: int, dim: int, dtype, device) -> int:
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.shape[2] != heads or c.shape[3] != dim or c.stride(3) != 1 or c.device != device:
            raise ValueError(f"{name} must be [pages, page_size, {heads}, {dim}] on {device} with unit last stride")
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache must have one shape and type")
    code = _CACHE_TYPE.get(k_cache.dtype)
    if code is None or (code != _lib.TYPE_E4M3 and k_cache.dtype != dtype):
        raise ValueError(f"the cache must be {dtype} or e4m3 (float8_e4m3fn or uint8), got {k_cache.dtype}")
    if not (1 <= k_cache.shape[0] <= _INT32_MAX and k_cache.shape[1] >= 1):
        raise ValueError("the cache needs at least one page of one token")
    return code


def _check_scale(name: str, t, heads: int, code: int, device) -> None:
    if t is None:
        return
    if code != _lib.TYPE_E4M3:
        raise ValueError(f"{name} goes with an e4m3 cache")
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != heads or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be fp32 [{heads}] on {device}")


_NO2, _NO3 = (0, 0), (0, 0, 0)


def _rotary(q, k, v, positions, table, sections, interleaved, pairing, inverse, q_out, k_out, caches, slots, k_scale,
            v_scale, status, stream, pdl_attr):
    """dg_rotary; returns (q_out, k_out), made here where they are True."""
    x = q if q is not None else k
    _need(x is not None and x.is_cuda, "q or k must be a CUDA tensor")
    _need(x.dim() == 3 and x.shape[0] >= 1 and x.dtype in _TYPE, "q and k must be bf16, fp16 or fp32 [tokens, heads, dim]")
    device, dtype = x.device, x.dtype
    tokens, _, dim = x.shape
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t is not None:
            _heads_of(name, t, tokens, dim, dtype, device)
    _need(table.dtype == torch.float32 and table.dim() == 2 and table.is_contiguous() and table.device == device,
          f"table must be a contiguous fp32 [max_position, rot] tensor on {device}")
    max_position, rot = table.shape
    _need(max_position >= 1 and 2 <= rot <= min(dim, _lib.MAX_ROT) and rot % 2 == 0,
          f"the table's width must be even and at most {min(dim, _lib.MAX_ROT)}")
    _need(pairing in _PAIRING, "pairing must be 'half' or 'adjacent'")
    axes, words = _axis_words(None if sections is None else tuple(sections), bool(interleaved), rot // 2)
    _need(positions.dtype in (torch.int32, torch.int64) and positions.device == device
          and positions.dim() in (1, 2) and positions.shape[-1] == tokens
          and (positions.stride(-1) == 1 or tokens == 1),
          f"positions must be int32 or int64 [{tokens}] or [axes, {tokens}] on {device}")
    position_stride = 0
    if positions.dim() == 2:
        _need(positions.shape[0] == axes, f"positions has {positions.shape[0]} axes, the sections {axes}")
        position_stride = positions.stride(0) if axes > 1 else 0
        _need(position_stride >= 0, "positions must not run backwards")
    _check_status(status)
    _check_same_device(device, status=status)
    heads = 0 if q is None else q.shape[1]
    kv_heads = 0 if k is None else k.shape[1]
    _need((q is None or heads >= 1) and (k is None or kv_heads >= 1), "q and k need at least one head")
    code = pages = page_size = 0
    k_cache = v_cache = None
    if caches is not None:
        k_cache, v_cache = caches
        _need(k.shape == v.shape, "k and v must have one shape")
        _need(dtype != torch.float32, "the cache write takes bf16 or fp16")
        code = _check_cache(k_cache, v_cache, kv_heads, dim, dtype, device)
        pages, page_size = k_cache.shape[:2]
        _check_ints("slots", slots, tokens, torch.int64)
        _check_same_device(device, slots=slots)
        _check_scale("k_scale", k_scale, kv_heads, code, device)
        _check_scale("v_scale", v_scale, kv_heads, code, device)
    for name, t, like in (("out_q", q_out, q), ("out_k", k_out, k)):
        if isinstance(t, torch.Tensor):
            _need(like is not None, f"{name} without its input")
            _heads_of(name, t, tokens, dim, dtype, device)
            _need(t.shape == like.shape, f"{name} must have its input's shape")
    with _on(device, stream) as handle:
        if q_out is True:
            q_out = torch.empty(q.shape, dtype=dtype, device=device)
        if k_out is True:
            k_out = torch.empty(k.shape, dtype=dtype, device=device)

        def two(t):
            return _NO2 if t is None else t.stride()[:2]

        def three(t):
            return _NO3 if t is None else t.stride()[:3]

        args = _lib.DgRotaryArgs(
            tokens, heads, kv_heads, dim, rot, _TYPE[dtype], code if caches is not None else _TYPE[dtype],
            _PAIRING[pairing], int(bool(inverse)), int(positions.dtype == torch.int64), max_position, page_size, pages,
            _addr(q), _addr(k), _addr(v), _addr(q_out), _addr(k_out), _addr(k_cache), _addr(v_cache),
            two(q), two(k), two(v), two(q_out), two(k_out), three(k_cache), three(v_cache),
            positions.data_ptr(), position_stride, _addr(slots), table.data_ptr(), _addr(k_scale), _addr(v_scale),
            _addr(status), words)
        _launch("dg_rotary", args, handle, pdl_attr)
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """rotary() where a gradient is wanted: a rotation's gradient is its
    inverse."""

    @staticmethod
    def forward(ctx, q, k, positions, table, kw):
        ctx.save_for_backward(positions, table)
        ctx.kw = kw
        return _rotary(q, k, None, positions, table, *kw[:3], kw[3], q is not None or None, k is not None or None, None,
                       None, None, None, *kw[4:])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, table = ctx.saved_tensors
        kw = ctx.kw
        dq, dk = (g if g is None or g.stride(-1) == 1 else g.contiguous() for g in (dq, dk))
        gq = gk = None
        if dq is not None or dk is not None:
            # On the stream and with the status of the moment, not of the forward pass.
            gq, gk = _rotary(dq, dk, None, positions, table, *kw[:3], not kw[3], dq is not None or None,
                             dk is not None or None, None, None, None, None, None, None, False)
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
    kw = (sections, interleaved, pairing, inverse, status, stream, pdl_attr)
    if torch.is_grad_enabled() and ((q is not None and q.requires_grad) or (k is not None and k.requires_grad)):
        _need(out_q is None and out_k is None, "out_q and out_k do not go with a gradient")
        return _Rotary.apply(q, k, positions, table, kw)
    return _rotary(q, k, None, positions, table, sections, interleaved, pairing, inverse,
                   out_q if out_q is not None else (True if q is not None else None),
                   out_k if out_k is not None else (True if k is not None else None),
                   None, None, None, None, status, stream, pdl_attr)


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
    _need(q is not None and k is not None and v is not None, "rotary_append takes q, k and v")
    return _rotary(q, k, v, positions, table, sections, interleaved, pairing, False,
                   out_q if out_q is not None else True, None, (k_cache, v_cache), slots, k_scale, v_scale, status,
                   stream, pdl_attr)[0]


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

_ATTENTION_WORKSPACES: dict = {}
_TICKET_BYTES = 1024


def attention_workspace(device="cuda") -> torch.Tensor:
    """A workspace for :func:`paged_attention` (about 5 MB, any arguments).
    Calls that can overlap on the GPU need one each."""
    nbytes = int(_lib.lib().dg_attention_workspace_bytes())
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    ws[:_TICKET_BYTES].zero_()               # the tickets; the rest is written before it is read
    return ws


def _stream_workspace(device, handle) -> torch.Tensor:
    # Kept per stream: calls on one stream run one after another.  A captured
    # graph may be replayed on any stream, so it gets its own, from its pool.
    if torch.cuda.is_current_stream_capturing():
        return attention_workspace(device)
    key = (device.index, handle)
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
    _need(q.is_cuda and q.dim() == 3 and q.dtype in (torch.bfloat16, torch.float16) and q.stride(2) == 1
          and q.shape[0] >= 1, "q must be bf16 or fp16 [batch >= 1, heads, dim] on a GPU with unit last stride")
    device, dtype = q.device, q.dtype
    batch, heads, dim = q.shape
    _need(k_cache.dim() == 4, "k_cache must be [pages, page_size, kv_heads, dim]")
    kv_heads = k_cache.shape[2]
    _need(kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0, "heads must be a multiple of the cache's heads")
    code = _check_cache(k_cache, v_cache, kv_heads, dim, dtype, device)
    unit = 16 if code == _lib.TYPE_E4M3 else 8
    _need(8 <= dim <= 256 and dim % unit == 0, f"dim must be a multiple of {unit}, at most 256")
    qs, ks, vs = q.stride(), k_cache.stride(), v_cache.stride()
    _need(qs[0] % 2 == 0 and qs[1] % 2 == 0 and q.data_ptr() % 4 == 0, "q must be 4-byte aligned with even strides")
    _need(ks[0] % unit == 0 and ks[1] % unit == 0 and ks[2] % unit == 0 and vs[0] % unit == 0 and vs[1] % unit == 0
          and vs[2] % unit == 0 and (k_cache.data_ptr() | v_cache.data_ptr()) % 16 == 0,
          "the caches must be 16-byte aligned, strides multiples of 16 bytes")
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch
          and block_table.shape[1] >= 1 and (block_table.stride(1) == 1 or block_table.shape[1] == 1)
          and block_table.device == device,
          f"block_table must be int32 [{batch}, width >= 1] on {device} with unit column stride")
    width = block_table.shape[1]
    table_stride = block_table.stride(0) if batch > 1 else width
    _need(table_stride >= width, "block_table's rows overlap")
    _check_ints("seq_lens", seq_lens, batch)
    _check_scale("k_scale", k_scale, kv_heads, code, device)
    _check_scale("v_scale", v_scale, kv_heads, code, device)
    _need(window is None or 1 <= window <= _INT32_MAX, "window must be at least 1")
    _need(softcap is None or 0.0 < softcap < float("inf"), "softcap must be positive")
    _check_status(status)
    _check_same_device(device, seq_lens=seq_lens, workspace=workspace, status=status)
    if out is not None:
        _heads_of("out", out, batch, dim, dtype, device)
        _need(out.shape == q.shape, "out must have q's shape")
    if q_out is not None or q_scales is not None:
        _need(q_out is not None and q_scales is not None, "q_out and q_scales go together")
        _need(dtype == torch.bfloat16 and dim % 128 == 0, "the quantised result takes bf16 and dim a multiple of 128")
        n = heads * dim
        _need(q_out.dtype in (torch.uint8, torch.float8_e4m3fn) and tuple(q_out.shape) == (batch, n)
              and q_out.is_contiguous() and q_out.device == device, f"q_out must be uint8 [{batch}, {n}], contiguous")
        _need(q_scales.dtype == torch.float32 and tuple(q_scales.shape) == (batch, n // 128)
              and q_scales.is_contiguous() and q_scales.device == device,
              f"q_scales must be fp32 [{batch}, {n // 128}], contiguous")
    if workspace is not None:
        _need(workspace.is_contiguous() and workspace.data_ptr() % 16 == 0
              and workspace.numel() * workspace.element_size() >= _lib.lib().dg_attention_workspace_bytes(),
              "workspace must come from attention_workspace()")
    with _on(device, stream) as handle:
        if out is None:
            out = torch.empty((batch, heads, dim), dtype=dtype, device=device)
        lse = torch.empty((batch, heads), dtype=torch.float32, device=device) if return_lse else None
        ws = workspace if workspace is not None else _stream_workspace(device, handle)
        args = _lib.DgAttentionArgs(
            batch, heads, kv_heads, dim, k_cache.shape[1], k_cache.shape[0], width, _TYPE[dtype], code, window or 0,
            dim ** -0.5 if scale is None else scale, softcap or 0.0, q.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), qs[:2], ks[:3], vs[:3], block_table.data_ptr(), table_stride, seq_lens.data_ptr(),
            _addr(k_scale), _addr(v_scale), out.data_ptr(), out.stride()[:2], _addr(lse), _addr(q_out),
            _addr(q_scales), ws.data_ptr(), ws.numel() * ws.element_size(), _addr(status))
        _launch("dg_paged_attention", args, handle, pdl_attr)
    return (out, lse) if return_lse else out
