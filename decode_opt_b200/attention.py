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
Nothing synchronises; every call can be captured in a CUDA graph.  Only
:func:`rotary` has a gradient, in q and k: a tensor that wants one elsewhere
raises ValueError.  torch.jit.trace, which would keep the results as constants,
is refused.  `stream` (default: the current one) takes a torch stream or a
cudaStream_t handle; outputs made here are allocated on it.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import importlib.util
import os
import struct
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib, build

__all__ = ["StepTables", "build_block_tables", "rope_table", "rotary", "rotary_append", "paged_attention",
           "attention_workspace"]

HOST_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_host.so")
_PAIRING = {"half": _lib.PAIR_HALF, "adjacent": _lib.PAIR_ADJACENT}


def _load():
    """The extension module that checks the tensors and makes the calls
    (csrc/dg_torch.cpp), bound to the library."""
    if not os.path.exists(HOST_PATH):
        raise RuntimeError(f"{HOST_PATH} is missing: build it with `python -m decode_opt_b200.build`")
    spec = importlib.util.spec_from_file_location("decode_opt_b200._host", HOST_PATH)
    host = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(host)
    if host.built_for != build.host_built_for():
        raise RuntimeError(f"{HOST_PATH} is the {host.built_for}: build it again with `python -m decode_opt_b200.build`")
    lib = _lib.lib()
    host.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
        "dg_build_block_tables", "dg_rotary", "dg_paged_attention", "dg_attention_workspace_bytes")))
    return host


_host = _load()


@contextlib.contextmanager
def _on(tensor, stream):
    """With the tensor's device and `stream` current."""
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise ValueError("the tensors must be CUDA tensors")
    s = torch.cuda.ExternalStream(stream, device=tensor.device) if isinstance(stream, int) else stream
    with torch.cuda.device(tensor.device), torch.cuda.stream(s):
        yield


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
    if stream is not None:
        with _on(context_lens, stream):
            return build_block_tables(context_lens, new_lens, free_pages, block_table, page_size, num_tokens,
                                      cursor=cursor, out=out, status=status, pdl_attr=pdl_attr)
    if out is None:
        return StepTables(*_host.build_block_tables(context_lens, new_lens, free_pages, block_table, page_size,
                                                    num_tokens, cursor, None, status, pdl_attr))
    _host.build_block_tables(context_lens, new_lens, free_pages, block_table, page_size, num_tokens, cursor,
                             (out.seq_lens, out.query_start, out.slots, out.positions, out.requests, out.cursor),
                             status, pdl_attr)
    return out


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------

def rope_table(max_position: int, rot: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos | sin of ``p * theta ** (-2i / rot)``, fp32 [max_position, rot]: made
    once, in 64 bits, for :func:`rotary` and :func:`rotary_append`."""
    if max_position < 1 or rot < 2 or rot % 2 != 0:
        raise ValueError("max_position >= 1 and an even rot >= 2")
    freq = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


@functools.lru_cache(maxsize=64)
def _axes(sections: Optional[Tuple[int, ...]], interleaved: bool, half: int):
    """(axes, each pair's axis packed as dg_rotary_args.axis_of) of `sections`."""
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
    if half > 16 * len(words):
        raise ValueError(f"the table's width must be at most {_lib.MAX_ROT}")
    for i, a in enumerate(axes):
        words[i // 16] |= a << (2 * (i % 16))
    return len(sections), struct.pack(f"@{len(words)}I", *words)


def _pairs(table, sections, interleaved, pairing):
    """(axes, packed axes, pairing code)."""
    code = _PAIRING.get(pairing)
    if code is None:
        raise ValueError("pairing must be 'half' or 'adjacent'")
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a tensor [max_position, rot]")
    axes, words = _axes(None if sections is None else tuple(sections), bool(interleaved), table.shape[1] // 2)
    return axes, words, code


class _Rotary(torch.autograd.Function):
    """rotary() where a gradient is wanted: a rotation's gradient is its
    inverse."""

    @staticmethod
    def forward(ctx, q, k, positions, table, pairs, inverse, status, pdl_attr):
        ctx.save_for_backward(positions, table)
        ctx.pairs, ctx.inverse = pairs, inverse
        ctx.set_materialize_grads(False)
        out = _host.rotary(q, k, None, positions, None, None, None, table, *pairs, inverse, None, None,
                           q is not None or None, k is not None or None, status, pdl_attr)
        ctx.mark_non_differentiable(*(y for y, wanted in zip(out, ctx.needs_input_grad)
                                      if y is not None and not wanted))
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, table = ctx.saved_tensors
        dq, dk = (None if g is None or not wanted else g if g.stride(-1) == 1 else g.contiguous()
                  for g, wanted in zip((dq, dk), ctx.needs_input_grad))
        gq = gk = None
        if dq is not None or dk is not None:
            gq, gk = _rotated(dq, dk, positions, table, ctx.pairs, not ctx.inverse, None, False)
        return gq, gk, None, None, None, None, None, None


def _untraced():
    """(The other calls look for themselves; rotary's gradient is an operation
    that a trace records.)"""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("torch.jit.trace cannot record rotary: its results would be constants of the trace")


def _tangent(x):
    """(x, None), or a forward-mode dual's primal and tangent."""
    if x is None:
        return None, None
    primal, tangent = forward_ad.unpack_dual(x)
    return primal, tangent if tangent is None or tangent.stride(-1) == 1 else tangent.contiguous()


def _rotated(q, k, positions, table, pairs, inverse, status, pdl_attr):
    """New rotated q and k, with what autograd wants of them: the map is
    linear, so that a tangent goes through it as the value does."""
    if forward_ad._current_level >= 0:
        (q, tq), (k, tk) = _tangent(q), _tangent(k)
        if tq is not None or tk is not None:
            values = _rotated(q, k, positions, table, pairs, inverse, status, pdl_attr)
            tangents = _rotated(tq, tk, positions, table, pairs, inverse, None, pdl_attr)
            return tuple(x if t is None else forward_ad.make_dual(x, t) for x, t in zip(values, tangents))
    if torch.is_grad_enabled() and ((q is not None and q.requires_grad) or (k is not None and k.requires_grad)):
        if table.requires_grad:
            raise ValueError("the table has no gradient")
        return _Rotary.apply(q, k, positions, table, pairs, inverse, status, pdl_attr)
    _untraced()
    return _host.rotary(q, k, None, positions, None, None, None, table, *pairs, inverse, None, None,
                        q is not None or None, k is not None or None, status, pdl_attr)


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
    back, which is also the gradient; the call is differentiable in q and k,
    backward and forward, without `out_q` and `out_k`.  These may be q and k
    themselves."""
    if stream is not None:
        with _on(q if q is not None else k, stream):
            return rotary(q, k, positions, table, sections=sections, interleaved=interleaved, pairing=pairing,
                          inverse=inverse, out_q=out_q, out_k=out_k, status=status, pdl_attr=pdl_attr)
    pairs = _pairs(table, sections, interleaved, pairing)
    if out_q is None and out_k is None:
        return _rotated(q, k, positions, table, pairs, inverse, status, pdl_attr)
    _untraced()
    return _host.rotary(q, k, None, positions, None, None, None, table, *pairs, inverse, None, None,
                        out_q if out_q is not None else (q is not None or None),
                        out_k if out_k is not None else (k is not None or None), status, pdl_attr)


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
    if stream is not None:
        with _on(q, stream):
            return rotary_append(q, k, v, positions, slots, k_cache, v_cache, table, sections=sections,
                                 interleaved=interleaved, pairing=pairing, k_scale=k_scale, v_scale=v_scale,
                                 out_q=out_q, status=status, pdl_attr=pdl_attr)
    if k_cache is None:
        raise ValueError("rotary_append takes the caches")
    return _host.rotary(q, k, v, positions, slots, k_cache, v_cache, table,
                        *_pairs(table, sections, interleaved, pairing), False, k_scale, v_scale,
                        True if out_q is None else out_q, None, status, pdl_attr)[0]


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def attention_workspace(device="cuda") -> torch.Tensor:
    """A workspace for :func:`paged_attention` (about 5 MB, any arguments).
    Calls that can overlap on the GPU need one each."""
    ws = torch.empty(int(_lib.lib().dg_attention_workspace_bytes()), dtype=torch.uint8, device=device)
    ws[:1024].zero_()                        # the tickets; the rest is written before it is read
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
    :func:`attention_workspace`; by default one is kept per stream (and host
    thread, on the per-thread default stream), and a call under capture gets
    its own, zeroed in the graph."""
    if stream is not None:
        with _on(q, stream):
            return paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale=scale, window=window,
                                   softcap=softcap, k_scale=k_scale, v_scale=v_scale, out=out, return_lse=return_lse,
                                   q_out=q_out, q_scales=q_scales, workspace=workspace, status=status,
                                   pdl_attr=pdl_attr)
    return _host.paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale, window, softcap, k_scale, v_scale,
                                 out, return_lse, q_out, q_scales, workspace, status, pdl_attr)
