"""The decode-attention operators, as cases to measure: block tables and slot maps from request lengths, rotary
positions with several axes (alone in both directions, and fused with the write into the paged key-value cache),
and the attention of one new token over that cache.

``run`` computes a case in its plain form -- elementary torch operations in 32 bits, rounded once -- or, where
``own`` is true, with the framework's operators on the same state.  ``exact`` gives the same outputs from the
definitions in 64 bits.
"""

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
_THETA = 1.0e6            # rotary base of long-context models
_MAX_POSITION = 131072    # rows of the cos/sin table


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One decode step of a small serving batch: latency only.
        {"name": "tables-decode", "kind": "tables", "batch": 16, "max_context": 4096, "prompts": 0, "max_new": 1,
         "page": 16},
        # Continuous batching: most requests decode one token, some bring a prompt; an odd batch.
        {"name": "tables-mixed", "kind": "tables", "batch": 501, "max_context": 8192, "prompts": 31, "max_new": 2048,
         "page": 64},
        # Offline processing: thousands of prompts admitted at once, 1.4 million tokens.
        {"name": "tables-prompts", "kind": "tables", "batch": 4096, "max_context": 0, "prompts": 4096,
         "max_new": 1024, "page": 16},
        # A decode step's rotation and cache write: eight tokens, one axis.
        {"name": "append-decode", "kind": "append", "tokens": 8, "pad": 0, "heads": 64, "kv_heads": 8, "dim": 128,
         "rot": 128, "type": "bf16", "cache": "bf16", "page": 16, "sections": "64", "interleaved": False,
         "pairing": "half"},
        # A prompt with images (time, height, width) into an 8-bit cache; an odd token count, padded to a graph's size.
        {"name": "append-image-e4m3", "kind": "append", "tokens": 4099, "pad": 61, "heads": 32, "kv_heads": 4,
         "dim": 128, "rot": 128, "type": "bf16", "cache": "e4m3", "page": 64, "sections": "16,24,24",
         "interleaved": False, "pairing": "half"},
        # A full prefill step of long prompts.
        {"name": "append-prefill", "kind": "append", "tokens": 32768, "pad": 0, "heads": 64, "kv_heads": 8,
         "dim": 128, "rot": 128, "type": "bf16", "cache": "bf16", "page": 16, "sections": "64",
         "interleaved": False, "pairing": "half"},
        # Training on video: forward and gradient, axes interleaved over the frequencies, half of each head rotated.
        {"name": "rotary-train-video", "kind": "rotary", "tokens": 12001, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 64, "type": "bf16", "sections": "12,10,10", "interleaved": True, "pairing": "adjacent"},
        # One request alone: the latency of a decode step's attention.
        {"name": "attention-one", "kind": "attention", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "bf16", "cache": "bf16", "page": 16, "max_len": 2049, "power": 0, "empty": 0, "window": 0, "cap": 0.0},
        # An ordinary serving batch: ragged lengths, grouped heads, some slots of the batch without a request.
        {"name": "attention-ragged", "kind": "attention", "batch": 61, "heads": 64, "kv_heads": 8, "dim": 128,
         "type": "bf16", "cache": "bf16", "page": 16, "max_len": 8191, "power": 2, "empty": 3, "window": 0, "cap": 0.0},
        # Every head its own keys, short heads, half precision, capped logits.
        {"name": "attention-heads-fp16", "kind": "attention", "batch": 33, "heads": 24, "kv_heads": 24, "dim": 64,
         "type": "fp16", "cache": "fp16", "page": 32, "max_len": 3000, "power": 1, "empty": 0, "window": 0, "cap": 30.0},
        # An 8-bit cache under 128 heads, a sliding window over the long requests.
        {"name": "attention-e4m3", "kind": "attention", "batch": 64, "heads": 128, "kv_heads": 8, "dim": 128,
         "type": "bf16", "cache": "e4m3", "page": 64, "max_len": 16384, "power": 1, "empty": 0, "window": 12000,
         "cap": 0.0},
        # Long contexts: 2.1 GB of cache read once.
        {"name": "attention-long", "kind": "attention", "batch": 32, "heads": 32, "kv_heads": 4, "dim": 128,
         "type": "bf16", "cache": "bf16", "page": 64, "max_len": 65536, "power": 1, "empty": 0, "window": 0, "cap": 0.0},
    ]


def _log_int(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("tables", "append", "rotary", "attention", "attention"))
    if kind == "tables":
        batch = _log_int(rng, 1, 4096)
        max_new = rng.choice((1, _log_int(rng, 2, 4096)))
        max_new = max(1, min(max_new, 4096 * 1024 // batch))
        page = rng.choice((1, 16, 24, 32, 64, 128))
        context = _log_int(rng, 1, min(32768, 4096 * 2048 * page // batch))     # tables of at most 8M entries or so
        return {"kind": kind, "batch": batch, "max_context": rng.choice((0, context)),
                "prompts": 0 if max_new == 1 else rng.randint(1, batch), "max_new": max_new, "page": page}
    dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8, 12, 16, 32))
    if kind == "attention":
        batch = _log_int(rng, 1, 160)
        cache = rng.choice(("bf16", "bf16", "fp16", "e4m3"))
        most = (32 * 65536 * 4 * 128) // (batch * kv_heads * dim)      # the largest listed case's padded cache
        most = min(most, (32 * 65536 * 4 * 128) // (batch * heads))    # and its bound on the plain form's scores
        max_len = _log_int(rng, 1, min(131072, most))
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "type": cache if cache != "e4m3" else rng.choice(("bf16", "fp16")), "cache": cache,
                "page": rng.choice((1, 16, 24, 32, 64, 128)), "max_len": max_len, "power": rng.choice((0, 1, 2)),
                "empty": rng.choice((0, 0, batch // 8)), "window": rng.choice((0, 0, _log_int(rng, 1, 32768))),
                "cap": rng.choice((0.0, 0.0, 30.0))}
    tokens = _log_int(rng, 1, min(65536, (32768 * 80 * 128) // ((heads + 2 * kv_heads) * dim)))
    rot = rng.choice((dim, dim, dim // 2))
    axes = rng.choice((1, 3))
    if axes == 1:
        sections = str(rot // 2)
    else:
        first = rot // 2 // 4
        second = (rot // 2 - first) // 2
        sections = "%d,%d,%d" % (first, second, rot // 2 - first - second)
    case = {"kind": kind, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "sections": sections, "interleaved": axes == 3 and rng.random() < 0.5,
            "pairing": rng.choice(("half", "half", "adjacent"))}
    if kind == "rotary":
        case["type"] = rng.choice(("bf16", "fp16", "fp32"))
        if case["type"] == "fp32":
            case["tokens"] = max(1, tokens // 4)
        else:
            case["tokens"] = max(1, tokens // 2)
        return case
    case["type"] = rng.choice(("bf16", "bf16", "fp16"))
    case["cache"] = rng.choice((case["type"], "e4m3"))
    case["page"] = rng.choice((1, 16, 24, 32, 64, 128))
    case["pad"] = rng.choice((0, rng.randint(1, 64)))
    return case


# ---------------------------------------------------------------------------
# Sizes that follow from a case alone
# ---------------------------------------------------------------------------

def _context_lens(case):
    b = case["batch"]
    return [case["max_context"] * (i + 1) // b for i in range(b)]


def _new_lens(case):
    """The first `prompts` requests bring 1 .. max_new tokens (a square law: many short ones), the others one."""
    n = case["prompts"]
    return [max(1, int(case["max_new"] * ((i + 1) / n) ** 2)) for i in range(n)] + [1] * (case["batch"] - n)


def _seq_lens(case):
    b = case["batch"]
    lens = [max(1, int(case["max_len"] * ((i + 1) / b) ** case["power"])) for i in range(b)]
    return [0] * case["empty"] + lens[case["empty"]:]


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["kind"] == "tables":
        b, page = case["batch"], case["page"]
        tokens = sum(_new_lens(case))
        pages = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(_context_lens(case), _new_lens(case)))
        # lengths, free pages and part-filled pages read; new entries, lengths, starts and 16 bytes a token written
        return {"bytes": 8 * b + 4 * pages + 4 * b + 4 * pages + 8 * b + 16 * tokens, "flops": 0}
    if case["kind"] in ("rotary", "append"):
        t, d, size = case["tokens"], case["dim"], _BYTES[case["type"]]
        axes = len(case["sections"].split(","))
        table = min(t, _MAX_POSITION) * case["rot"] * 4
        rotated = (case["heads"] + case["kv_heads"]) * t
        if case["kind"] == "rotary":   # q, k and their gradients, in and out
            return {"bytes": 4 * rotated * d * size + table + axes * t * 8, "flops": 2 * rotated * case["rot"] * 3}
        q = (t + case["pad"]) * case["heads"] * d * size
        kv = 2 * t * case["kv_heads"] * d
        return {"bytes": 2 * q + kv * size + kv * _BYTES[case["cache"]] + table + (t + case["pad"]) * (8 + 8 * axes),
                "flops": rotated * case["rot"] * 3}
    lens = _seq_lens(case)
    if case["window"]:
        lens = [min(n, case["window"]) for n in lens]
    b, h, d = case["batch"], case["heads"], case["dim"]
    kv = 2 * sum(lens) * case["kv_heads"] * d * _BYTES[case["cache"]]
    return {"bytes": kv + 2 * b * h * d * _BYTES[case["type"]] + 4 * b * h + 4 * b
            + 4 * sum(_pages(n, case["page"]) for n in lens), "flops": 4 * sum(lens) * h * d}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _axes_of(case):
    """The axis of each frequency: the sections one after another, or dealt in turn while an axis has some left."""
    left = [int(s) for s in case["sections"].split(",")]
    if not case["interleaved"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    axes = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                axes.append(a)
    return axes


def _shuffled(values, g, dtype=torch.int32):
    order = torch.randperm(len(values), generator=g, device="cuda")
    return torch.tensor(values, dtype=dtype, device="cuda")[order]


def _rotary_table(rot):
    freq = _THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(_MAX_POSITION, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _positions(tokens, axes, g):
    """Where a prompt's tokens stand: text counts on all axes at once; pictures of 16 x 16 patches stand still in
    time and count rows and columns."""
    start = int(torch.randint(0, _MAX_POSITION - tokens - 64, (1,), generator=g, device="cuda"))
    t = torch.arange(tokens, dtype=torch.int64, device="cuda")
    if axes == 1:
        return (start + t)[None]
    image, inside = t // 256, t % 256
    text = image % 4 == 3
    base = start + image * 16
    time = torch.where(text, start + t, base)
    row = torch.where(text, start + t, base + inside // 16)
    column = torch.where(text, start + t, base + inside % 16)
    return torch.stack([time, row, column])


def _prepare_tables(case, g):
    page, b = case["page"], case["batch"]
    context, new = _context_lens(case), _new_lens(case)
    order = torch.randperm(b, generator=g, device="cuda")
    context = torch.tensor(context, dtype=torch.int32, device="cuda")[order]
    new = _shuffled(new, g)
    held = (context + page - 1) // page
    most = (case["max_context"] + case["max_new"] + page - 1) // page + 1
    pool = torch.randperm(b * most, generator=g, device="cuda").to(torch.int32)
    mine = torch.arange(most, device="cuda")[None] < held[:, None]
    table = torch.where(mine, pool[:b * most].view(b, most), -1)
    free = pool.view(b, most)[~mine]
    total = sum(_new_lens(case))
    return {"context": context, "new": new, "table": table.contiguous(), "free": free.contiguous(), "page": page,
            "tokens": -(-total // 64) * 64}


def _prepare_rotary(case, g):
    t, d, dtype = case["tokens"], case["dim"], _TYPES[case["type"]]
    sections = tuple(int(s) for s in case["sections"].split(","))
    rnd = lambda h: torch.randn(t, h, d, generator=g, device="cuda").to(dtype)  # noqa: E731
    return {"q": rnd(case["heads"]), "k": rnd(case["kv_heads"]), "dq": rnd(case["heads"]), "dk": rnd(case["kv_heads"]),
            "positions": _positions(t, len(sections), g), "table": _rotary_table(case["rot"]), "sections": sections,
            "axes": torch.tensor(_axes_of(case), device="cuda")}


def _prepare_append(case, g):
    live, d, page, h, hk = case["tokens"], case["dim"], case["page"], case["heads"], case["kv_heads"]
    t = live + case["pad"]
    dtype, cache = _TYPES[case["type"]], _TYPES[case["cache"]]
    sections = tuple(int(s) for s in case["sections"].split(","))
    qkv = torch.randn(t, (h + 2 * hk) * d, generator=g, device="cuda").to(dtype)   # as a fused projection leaves it
    pages = _pages(live, page) + 3                                                 # the last page is in no table
    order = torch.randperm(pages - 1, generator=g, device="cuda")
    tok = torch.arange(t, device="cuda")
    at = (tok + page // 2).clamp(max=_pages(live + page // 2, page) * page - 1)
    slots = torch.where(tok < live, order[at // page] * page + at % page, -1)
    old = lambda: torch.randn(pages, page, hk, d, generator=g, device="cuda").to(cache)  # noqa: E731
    state = {"q": qkv[:, :h * d].view(t, h, d), "k": qkv[:, h * d:(h + hk) * d].view(t, hk, d),
             "v": qkv[:, (h + hk) * d:].view(t, hk, d), "positions": _positions(t, len(sections), g), "slots": slots,
             "k_cache": old(), "v_cache": old(), "table": _rotary_table(case["rot"]), "sections": sections,
             "axes": torch.tensor(_axes_of(case), device="cuda"), "k_scale": None, "v_scale": None}
    if case["cache"] == "e4m3":
        state["k_scale"] = torch.rand(hk, generator=g, device="cuda") * 0.02 + 0.01
        state["v_scale"] = torch.rand(hk, generator=g, device="cuda") * 0.02 + 0.01
    return state


def _prepare_attention(case, g):
    b, h, hk, d, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype, cache = _TYPES[case["type"]], _TYPES[case["cache"]]
    lens = _seq_lens(case)
    held = [_pages(n, page) for n in lens]
    pages = sum(held) + 1
    order = torch.randperm(b, generator=g, device="cuda")
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")[order]
    held = torch.tensor(held, dtype=torch.int32, device="cuda")[order]
    width = max(1, _pages(case["max_len"], page))
    pool = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    mine = torch.arange(width, device="cuda")[None] < held[:, None]
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    table[mine] = pool[:int(held.sum())]
    state = {"table": table, "seq_lens": seq_lens, "k_scale": None, "v_scale": None, "scale": d ** -0.5}
    spread = 1.0
    if case["cache"] == "e4m3":
        state["k_scale"] = torch.rand(hk, generator=g, device="cuda") * 0.02 + 0.01
        state["v_scale"] = torch.rand(hk, generator=g, device="cuda") * 0.02 + 0.01
        spread = 50.0
    # From flat logits to heads that look at a few tokens.
    sharp = torch.linspace(0.3, 3.0, h, device="cuda")[None, :, None]
    state["q"] = (torch.randn(b, h, d, generator=g, device="cuda") * sharp).to(dtype)
    fill = lambda: (torch.randn(pages, page, hk, d, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
                    * spread).clamp(-448, 448).to(cache)
    state["k_cache"], state["v_cache"] = fill(), fill()
    return state


_PREPARE = {"tables": _prepare_tables, "rotary": _prepare_rotary, "append": _prepare_append,
            "attention": _prepare_attention}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = _PREPARE[case["kind"]](case, g)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _tables(s):
    if own:
        import decode_opt_b200 as dg
        p = dg.build_block_tables(s["context"], s["new"], s["free"], s["table"], s["page"], s["tokens"])
        return {"table": s["table"], "seq_lens": p.seq_lens, "query_start": p.query_start, "slots": p.slots,
                "positions": p.positions, "requests": p.requests, "cursor": p.cursor}
    page, context, new, table, free = s["page"], s["context"], s["new"], s["table"], s["free"]
    lens = context + new
    held, need = (context + page - 1) // page, (lens + page - 1) // page
    taken = torch.cumsum(need - held, 0, dtype=torch.int64)
    column = torch.arange(table.shape[1], device="cuda")[None]
    source = (taken - (need - held))[:, None] + column - held[:, None]
    fresh = (column >= held[:, None]) & (column < need[:, None])
    table = torch.where(fresh, free[source.clamp(0, free.numel() - 1)], table)
    start = torch.cat([new.new_zeros(1), torch.cumsum(new, 0, dtype=torch.int32)])
    token = torch.arange(s["tokens"], dtype=torch.int32, device="cuda")
    request = torch.searchsorted(start[1:], token, right=True).clamp(max=new.numel() - 1)
    live = token < start[-1]
    position = context[request] + token - start[request]
    entry = table[request, (position // page).clamp(max=table.shape[1] - 1).long()].long()
    slot = torch.where(live, entry * page + position % page, -1)
    return {"table": table, "seq_lens": lens, "query_start": start, "slots": slot,
            "positions": torch.where(live, position, 0), "requests": torch.where(live, request, -1).to(torch.int32),
            "cursor": taken[-1:].to(torch.int32)}


def _turn(x, cos, sin, case):
    """x [T, H, D] with its first `rot` values rotated, in x's floating type of computation."""
    rot = case["rot"]
    cos, sin = cos[:, None], sin[:, None]
    if case["pairing"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], dim=-1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), x[..., rot:]], dim=-1)


def _cos_sin(s):
    half = s["case"]["rot"] // 2
    where = s["positions"][s["axes"]]                       # [rot/2, T]
    pair = torch.arange(half, device="cuda")[:, None]
    return s["table"][where, pair].T, s["table"][where, half + pair].T


def _rotary(s):
    c = s["case"]
    if own:
        import decode_opt_b200 as dg
        kw = dict(sections=s["sections"], interleaved=c["interleaved"], pairing=c["pairing"])
        q, k = dg.rotary(s["q"], s["k"], s["positions"], s["table"], **kw)
        dq, dk = dg.rotary(s["dq"], s["dk"], s["positions"], s["table"], inverse=True, **kw)
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    cos, sin = _cos_sin(s)
    return {n: _turn(s[n].float(), cos, -sin if n[0] == "d" else sin, c).to(s[n].dtype) for n in ("q", "k", "dq", "dk")}


def _store(cache, slots, x, scale):
    """cache [pages, page, H, D] with rows x [T, H, D] at the slots; those below 0 go to the pool's last row, which
    is in no table."""
    x = x if scale is None else (x / scale[None, :, None]).clamp(-448, 448)
    flat = cache.view(-1, *cache.shape[2:])
    where = torch.where(slots < 0, flat.shape[0] - 1, slots)
    if cache.dtype == torch.float8_e4m3fn:
        flat.view(torch.uint8)[where] = x.to(cache.dtype).view(torch.uint8)
    else:
        flat[where] = x.to(cache.dtype)
    return cache[:-1]


def _append(s):
    c = s["case"]
    if own:
        import decode_opt_b200 as dg
        q = dg.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
                             s["table"], sections=s["sections"], interleaved=c["interleaved"], pairing=c["pairing"],
                             k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"q": q, "k_cache": s["k_cache"][:-1], "v_cache": s["v_cache"][:-1]}
    cos, sin = _cos_sin(s)
    q = _turn(s["q"].float(), cos, sin, c).to(s["q"].dtype)
    return {"q": q, "k_cache": _store(s["k_cache"], s["slots"], _turn(s["k"].float(), cos, sin, c), s["k_scale"]),
            "v_cache": _store(s["v_cache"], s["slots"], s["v"].float(), s["v_scale"])}


def _gathered(cache, table, scale, dtype):
    """The requests' rows of a cache, padded: [B, Hk, width * page, D]."""
    b, width = table.shape
    bits = torch.uint8 if cache.dtype == torch.float8_e4m3fn else cache.dtype
    rows = cache.view(bits)[table.clamp(min=0).long()].view(cache.dtype).to(dtype)       # [B, width, page, Hk, D]
    rows = rows.view(b, width * cache.shape[1], *cache.shape[2:]).transpose(1, 2)
    return rows if scale is None else rows * scale.to(dtype)[None, :, None, None]


def _attention(s):
    c = s["case"]
    if own:
        import decode_opt_b200 as dg
        out, lse = dg.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], scale=s["scale"],
                                      window=c["window"] or None, softcap=c["cap"] or None, k_scale=s["k_scale"],
                                      v_scale=s["v_scale"], return_lse=True)
        return {"out": out, "lse": lse}
    b, h, d = s["q"].shape
    hk = s["k_cache"].shape[2]
    lens = s["seq_lens"][:, None, None, None]
    q = s["q"].float().view(b, hk, h // hk, d)
    k = _gathered(s["k_cache"], s["table"], s["k_scale"], torch.float32)
    logit = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    del k
    if c["cap"]:
        logit = c["cap"] * torch.tanh(logit / c["cap"])
    token = torch.arange(logit.shape[-1], device="cuda")
    seen = token < lens
    if c["window"]:
        seen = seen & (token >= lens - c["window"])
    logit = torch.where(seen, logit, -torch.inf)
    top = logit.amax(-1, keepdim=True).clamp(min=-3.0e38)
    p = torch.exp(logit - top)
    total = p.sum(-1, keepdim=True)
    v = _gathered(s["v_cache"], s["table"], s["v_scale"], torch.float32)
    out = torch.matmul(p, v) / total
    out = torch.where(lens > 0, out, 0.0)
    lse = torch.where(lens > 0, top + torch.log(total), -torch.inf)
    return {"out": out.view(b, h, d).to(s["q"].dtype), "lse": lse.view(b, h)}


_RUN = {"tables": _tables, "rotary": _rotary, "append": _append, "attention": _attention}


def run(state):
    return _RUN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_turn(x, positions, axes, case, sign):
    """Each pair as a complex number, turned by its angle."""
    rot = case["rot"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    angle = positions[axes].T.double() * torch.exp(-2.0 * i / rot * torch.log(torch.tensor(_THETA, dtype=torch.float64)))
    turn = torch.polar(torch.ones_like(angle), sign * angle)[:, None]
    x = x.double()
    out = x.clone()
    if case["pairing"] == "half":
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
        out[..., :rot // 2], out[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.view_as_complex(x[..., :rot].contiguous().unflatten(-1, (rot // 2, 2))) * turn
        out[..., :rot] = torch.view_as_real(z).flatten(-2)
    return out


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return {n: _exact_turn(s[n], s["positions"], s["axes"], case, -1.0 if n[0] == "d" else 1.0)
                for n in ("q", "k", "dq", "dk")}
    if case["kind"] == "append":
        live = s["slots"] >= 0
        result = {"q": _exact_turn(s["q"], s["positions"], s["axes"], case, 1.0)}
        rows = {"k_cache": _exact_turn(s["k"], s["positions"], s["axes"], case, 1.0), "v_cache": s["v"].double()}
        for name, x in rows.items():
            cache, scale = s[name].double(), s[name[0] + "_scale"]
            x = x if scale is None else x / scale.double()[None, :, None]
            cache.view(-1, *cache.shape[2:])[s["slots"][live]] = x[live]
            result[name] = cache[:-1]
        return result
    q, page = s["q"].double(), case["page"]
    b, h, d = q.shape
    hk = case["kv_heads"]
    out = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h), -torch.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["seq_lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda")
        slot = s["table"][r].long()[at // page] * page + at % page
        for head in range(hk):
            rows = []
            for name in ("k", "v"):
                x = s[name + "_cache"].view(-1, hk, d)[:, head]
                x = (x.view(torch.uint8)[slot].view(x.dtype) if case["cache"] == "e4m3" else x[slot]).double()
                rows.append(x if s[name + "_scale"] is None else x * s[name + "_scale"][head].double())
            of = slice(head * (h // hk), (head + 1) * (h // hk))
            logit = (q[r, of] @ rows[0].T) * s["scale"]
            if case["cap"]:
                logit = case["cap"] * torch.tanh(logit / case["cap"])
            lse[r, of] = torch.logsumexp(logit, -1)
            out[r, of] = torch.softmax(logit, -1) @ rows[1]
    return {"out": out, "lse": lse}
