"""The attention half of a decode layer, from the framework's operators:

    x [M, hidden] bf16
      -> e4m3 + block scales           quantize_activation
      -> q, k, v                       fp8_decode_gemm, one product
      -> rotated q; k, v in the cache  rotary_append
      -> attention over the cache      paged_attention, quantised as it is written
      -> [M, hidden] bf16              fp8_decode_gemm (the output projection)

for M = 1 .. 128 requests that bring one token each, over a paged cache whose
bookkeeping build_block_tables makes on the GPU once per step for all layers.

    python -m decode_opt_b200.decode_layer --requests 32 --context 4096 --steps 64

runs it with random weights as a captured CUDA graph and prints the time of a
step and of its parts.
"""

from __future__ import annotations

import argparse
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

import decode_opt_b200 as dg


@dataclass(frozen=True)
class LayerShape:
    hidden: int
    heads: int
    kv_heads: int
    head_dim: int
    sections: Optional[Sequence[int]] = None     # rotary axes, see dg.rotary
    window: Optional[int] = None

    @property
    def q_width(self) -> int:
        return self.heads * self.head_dim

    @property
    def qkv_width(self) -> int:
        return (self.heads + 2 * self.kv_heads) * self.head_dim


class PagedCache:
    """One layer's key-value cache: [pages, page_size, kv_heads, head_dim], bf16
    or e4m3 with a scale per head."""

    def __init__(self, shape: LayerShape, pages: int, page_size: int, dtype=torch.bfloat16, k_scale=None, v_scale=None,
                 device="cuda"):
        size = (pages, page_size, shape.kv_heads, shape.head_dim)
        self.k = torch.zeros(size, dtype=torch.float32 if dtype.itemsize == 1 else dtype, device=device).to(dtype)
        self.v = self.k.clone()
        self.k_scale, self.v_scale = k_scale, v_scale


class DecodeAttention:
    """The layer's weights, prepacked once, and its step.

    ``w_qkv`` e4m3 [qkv_width, hidden] and ``w_out`` e4m3 [hidden, q_width]
    (uint8) come with the GEMM's block scales [ceil(N / 128), K / 128]; hidden
    and q_width are multiples of 128.  The quantised attention output needs a
    head_dim that is a multiple of 128; other heads are quantised by a kernel
    of their own."""

    def __init__(self, shape: LayerShape, w_qkv, qkv_scales, w_out, out_scales, batch: int):
        if shape.hidden % 128 != 0 or shape.q_width % 128 != 0:
            raise ValueError("hidden and heads * head_dim must be multiples of 128")
        if tuple(w_qkv.shape) != (shape.qkv_width, shape.hidden) or tuple(w_out.shape) != (shape.hidden, shape.q_width):
            raise ValueError("w_qkv must be [qkv_width, hidden] and w_out [hidden, q_width]")
        self.shape = shape
        layout = dg.LAYOUT_PACKED_SWIZZLED
        self.qkv_config = dg.default_config(batch, shape.qkv_width, shape.hidden, layout=layout)
        self.out_config = dg.default_config(batch, shape.hidden, shape.q_width, layout=layout)
        self.w_qkv = dg.prepack_weight(w_qkv, self.qkv_config.packed_rows, layout)
        self.w_out = dg.prepack_weight(w_out, self.out_config.packed_rows, layout)
        self.qkv_scales, self.out_scales = qkv_scales, out_scales

    def step(self, x, step: "dg.StepTables", block_table, cache: PagedCache, table, workspace=None) -> torch.Tensor:
        """One token of each request: x [M, hidden] bf16 -> [M, hidden] bf16, on
        the current stream.  `step` is of the same M requests, one new token
        each, without padding.

        Steps may run on several streams at once.  `workspace` is that of
        :func:`dg.paged_attention`: by default its own per stream and per
        captured call.  One from :func:`dg.attention_workspace` saves a captured
        step the zeroing; steps that share it must not overlap."""
        s, m = self.shape, x.shape[0]
        act, act_scales = dg.quantize_activation(x, stream=torch.cuda.current_stream(x.device))
        qkv = dg.fp8_decode_gemm(act, act_scales, self.w_qkv, self.qkv_scales, config=self.qkv_config, n=s.qkv_width)
        qkv = qkv.view(m, s.heads + 2 * s.kv_heads, s.head_dim)
        q, k, v = qkv.split_with_sizes((s.heads, s.kv_heads, s.kv_heads), 1)
        q = dg.rotary_append(q, k, v, step.positions, step.slots, cache.k, cache.v, table, sections=s.sections,
                             k_scale=cache.k_scale, v_scale=cache.v_scale)
        kw = dict(window=s.window, k_scale=cache.k_scale, v_scale=cache.v_scale, workspace=workspace)
        if s.head_dim % 128 == 0:
            act = torch.empty((m, s.q_width), dtype=torch.uint8, device=x.device)
            act_scales = torch.empty((m, s.q_width // 128), dtype=torch.float32, device=x.device)
            dg.paged_attention(q, cache.k, cache.v, block_table, step.seq_lens, q_out=act, q_scales=act_scales, **kw)
        else:
            out = dg.paged_attention(q, cache.k, cache.v, block_table, step.seq_lens, **kw)
            act, act_scales = dg.quantize_activation(out.view(m, s.q_width),
                                                     stream=torch.cuda.current_stream(x.device))
        return dg.fp8_decode_gemm(act, act_scales, self.w_out, self.out_scales, config=self.out_config, n=s.hidden)


def random_layer(shape: LayerShape, batch: int, seed: int = 0, device="cuda") -> DecodeAttention:
    """Random weights whose products keep values near 1."""
    g = torch.Generator(device=device).manual_seed(seed)

    def weight(n, k):
        w = torch.randn(n, k, generator=g, device=device).to(torch.float8_e4m3fn).view(torch.uint8)
        return w, torch.full((-(-n // 128), k // 128), k ** -0.5, device=device)
    return DecodeAttention(shape, *weight(shape.qkv_width, shape.hidden), *weight(shape.hidden, shape.q_width), batch)


def free_list(block_table, held: int):
    """The pages of the table's columns from `held` on, as a free list of its
    own: a view of the table would be overwritten as the table is filled."""
    return block_table[:, held:].flatten().clone()


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--context", type=int, default=4096, help="tokens a request has in the cache")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--hidden", type=int, default=7168)
    ap.add_argument("--heads", type=int, default=64)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--page-size", type=int, default=64)
    ap.add_argument("--e4m3-cache", action="store_true")
    o = ap.parse_args(argv)
    if not 1 <= o.requests <= 128:
        ap.error("--requests must be 1 .. 128")
    shape = LayerShape(o.hidden, o.heads, o.kv_heads, o.head_dim)
    m, dev = o.requests, torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    layer = random_layer(shape, m)
    width = -(-(o.context + o.steps + 8) // o.page_size)
    held = -(-o.context // o.page_size)
    pool = torch.randperm(m * width, device=dev).to(torch.int32)
    block_table = pool.view(m, width).clone()
    free, cursor = free_list(block_table, held), torch.zeros(1, dtype=torch.int32, device=dev)
    scales = [torch.full((o.kv_heads,), 0.02, device=dev) if o.e4m3_cache else None for _ in range(2)]
    cache = PagedCache(shape, m * width, o.page_size, torch.float8_e4m3fn if o.e4m3_cache else torch.bfloat16, *scales)
    table = dg.rope_table(o.context + o.steps + 8, o.head_dim)
    lens = torch.full((m,), o.context, dtype=torch.int32, device=dev)
    new = torch.ones(m, dtype=torch.int32, device=dev)
    x = torch.randn(m, o.hidden, device=dev).bfloat16()
    workspace = dg.attention_workspace(dev)

    def once():
        t = dg.build_block_tables(lens, new, free, block_table, o.page_size, m, cursor=cursor)
        y = layer.step(x, t, block_table, cache, table, workspace)
        x.copy_(y)
        lens.copy_(t.seq_lens)
        cursor.copy_(t.cursor)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()                               # workspaces and lazily loaded kernels
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            once()
        for _ in range(3):
            graph.replay()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record(side)
        for _ in range(o.steps):
            graph.replay()
        end.record(side)
        side.synchronize()
    us = begin.elapsed_time(end) * 1e3 / o.steps
    kv = 2 * m * o.context * o.kv_heads * o.head_dim * cache.k.element_size()
    weights = shape.qkv_width * shape.hidden + shape.hidden * shape.q_width
    print(f"{m} requests, {o.context} tokens each: {us:.1f} us a step (block tables and one layer's attention half); "
          f"cache {kv / 1e6:.1f} MB, weights {weights / 1e6:.1f} MB, {(kv + weights) / us / 1e3:.0f} GB/s")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
