"""Operators of a serving step over the NVFP4 paged cache, as a user calls them, with a plain form of each.

Three operators that one step of long, image-bearing sequences calls in a row: ``extend_pages`` (block
tables, slot map and positions of the step's tokens from the requests' lengths, with ``trim_pages``
for what falls out of a window), rotary positions with several axes (``apply_rope`` and
``write_nvfp4_rope_rotated`` with positions [axes, tokens]) and ``mla_prefill`` with a sliding window
and first tokens that stay visible.

With ``own`` false, ``run`` computes them in elementary torch operations; with ``own`` true it makes
the framework's calls on the same inputs.
"""
import math
import random

import torch

own = False

LATENT, ROPE, ROW = 512, 64, 288
SCALE = 1.0 / 24.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of 16 sequences, one token each: latency counts
        {"name": "pages_decode", "op": "pages", "kind": "step", "requests": 16, "slots": 16, "context": 8192, "new": 1,
         "pages": 4096, "page": 64, "width": 2048, "pad": 0, "mix": 1},
        # a speculative step: up to 5 draft tokens each, the tokens that were not accepted taken back first
        {"name": "pages_spec", "op": "pages", "kind": "spec", "requests": 100, "slots": 128, "context": 2000, "new": 5,
         "pages": 15000, "page": 16, "width": 200, "pad": 12, "mix": 2},
        # 16 chunks of 2,048 tokens in a pool of about 2.7 million
        {"name": "pages_chunks", "op": "pages", "kind": "step", "requests": 16, "slots": 64, "context": 131072, "new": 2048,
         "pages": 42405, "page": 64, "width": 4688, "pad": 0, "mix": 3},
        # prompts of many requests placed at once, and what lies behind their window given back
        {"name": "pages_window", "op": "pages", "kind": "window", "requests": 480, "slots": 512, "context": 0, "new": 2000,
         "pages": 42405, "page": 64, "width": 256, "pad": 100, "mix": 4, "window": 512, "sinks": 4},
        # time, height and width on the queries of a decode step
        {"name": "axes_decode", "op": "rope", "tokens": 16, "heads": 64, "dim": 576, "rotary": 64, "offset": 512,
         "interleaved": True, "inverse": False, "dtype": "bf16", "positions": 131072, "axes": 3, "dealt": False},
        # a prompt of images, whole heads turned, the axes dealt to the pairs in turn
        {"name": "axes_images", "op": "rope", "tokens": 8192, "heads": 32, "dim": 128, "rotary": 128, "offset": 0,
         "interleaved": False, "inverse": False, "dtype": "bf16", "positions": 8192, "axes": 3, "dealt": True},
        # the gradient, two axes, an odd number of tokens
        {"name": "axes_backward", "op": "rope", "tokens": 2049, "heads": 20, "dim": 192, "rotary": 64, "offset": 128,
         "interleaved": True, "inverse": True, "dtype": "fp32", "positions": 8192, "axes": 2, "dealt": False},
        # the write seam of 16 chunks of 2,048 tokens
        {"name": "axes_write", "op": "write", "tokens": 32768, "heads": 16, "q_dim": 192, "pages": 4096, "page": 64,
         "interleaved": True, "positions": 131072, "axes": 3, "dealt": True},
        # a speculative step over short windows, odd lengths, no rope part
        {"name": "window_short", "op": "window", "batch": 3, "new": 7, "context": 777, "heads": 16, "page": 64, "rope": False,
         "decodes": 1, "mix": 5, "window": 128, "sinks": 4, "trim": False},
        # single tokens of 16 sequences whose old pages are gone
        {"name": "window_single", "op": "window", "batch": 16, "new": 1, "context": 8192, "heads": 64, "page": 64, "rope": True,
         "decodes": 16, "mix": 3, "window": 1024, "sinks": 4, "trim": True},
        # a mixed step: chunks among single tokens
        {"name": "window_mixed", "op": "window", "batch": 8, "new": 777, "context": 8192, "heads": 32, "page": 16, "rope": True,
         "decodes": 5, "mix": 4, "window": 512, "sinks": 100, "trim": True},
        # a 2,048-token chunk of a long prompt, 64 heads: compute-bound
        {"name": "window_chunk", "op": "window", "batch": 1, "new": 2048, "context": 131072, "heads": 64, "page": 64,
         "rope": True, "decodes": 0, "mix": 2, "window": 4096, "sinks": 64, "trim": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "pages", "rope", "write", "window", "window"])
    if op == "pages":
        kind = rng.choice(["step", "spec", "window"])
        page, requests = rng.choice([16, 64, 128]), _log(rng, 1, 400)
        context = 0 if kind == "window" else _log(rng, 1, 8000)
        new = rng.randint(1, 8) if kind == "spec" else _log(rng, 1, 30000 // requests + 1)
        width = (context + 2 * new) // page + rng.randint(2, 100)
        return {"op": op, "kind": kind, "requests": requests, "slots": requests + rng.randint(0, 40), "context": context,
                "new": new, "pages": requests * width + rng.randint(0, 4000), "page": page, "width": width,
                "pad": rng.randint(0, 64), "mix": rng.randint(0, 1 << 20), "window": _log(rng, 1, 4096),
                "sinks": rng.choice([0, 1, 4, 64, 100])}
    axes, dealt = rng.randint(2, 4), rng.random() < 0.5
    if op == "rope":
        rotary = rng.choice([16, 32, 64, 128])
        dim, offset = rng.choice([(576, 576 - rotary), (128, 0), (192, 192 - rotary)])
        heads = rng.randint(1, 64)
        return {"op": op, "tokens": _log(rng, 1, 8192 * 32 * 128 // (2 * heads * dim)), "heads": heads, "dim": dim,
                "rotary": rotary, "offset": offset, "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.3,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "positions": rng.choice([8192, 131072]),
                "axes": axes, "dealt": dealt}
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 30000), "heads": rng.randint(1, 16), "q_dim": rng.choice([64, 192]),
                "pages": rng.randint(1000, 2000) * 64 // 16, "page": rng.choice([16, 64]),
                "interleaved": rng.random() < 0.5, "positions": rng.choice([8192, 131072]), "axes": axes, "dealt": dealt}
    context = _log(rng, 1, 65536)
    batch, window, sinks = rng.randint(1, 8), _log(rng, 1, 4096), rng.choice([0, 1, 4, 16, 64, 100, 200])
    heads = rng.choice([1, 4, 16, 20, 32, 64, 128])
    wide = min(window, context) + sinks                        # scores: batch x new x heads x (wide + new)
    most = min(int((math.sqrt(wide * wide + 4 * 600000000 / (batch * heads)) - wide) / 2), 131072 // (batch * heads))
    return {"op": op, "batch": batch, "new": _log(rng, 1, max(1, min(context, most, 2048))), "context": context, "heads": heads,
            "page": rng.choice([16, 64, 128]), "rope": rng.random() < 0.7, "decodes": rng.randint(0, batch),
            "mix": rng.randint(0, 1 << 20), "window": window, "sinks": sinks, "trim": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cos_sin(positions, rotary, factor=4.0):
    """cos | sin of every position, [positions, rotary] float32: long contexts by scaled frequencies."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary) / factor
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _pair_axes(case, rotary):
    """The axis of each rotated pair: in sections, or dealt in turn."""
    half, n = rotary // 2, case["axes"]
    return tuple(i % n for i in range(half)) if case["dealt"] else tuple(min(i * n // half, n - 1) for i in range(half))


def _axis_positions(g, case):
    """[axes, tokens]: text, whose axes agree, between images (a time, then rows and columns of a grid)."""
    T, most = case["tokens"], case["positions"]
    t = torch.arange(T, device="cuda")
    side = 24
    start = torch.randint(0, most - T - side, (1,), generator=g, device="cuda") if most > T + side else 0
    at = t % (2 * side * side)                           # half of the tokens are text
    image = at >= side * side
    base = start + t - torch.where(image, at - side * side, 0)
    cell = (at - side * side).clamp_min(0)
    axes = [base, base + cell // side, base + cell % side, base + cell // (side * 4)]
    pos = torch.stack([torch.where(image, a, base) for a in axes[: case["axes"]]])
    return (pos % most).int()


def _pack_nvfp4(x):
    """[n, 512] values -> 288-byte rows: e2m1 codes and one e4m3 scale for 16 of them."""
    v = x.float().view(-1, 32, 16)
    s = (v.abs().amax(2) / 6.0).clamp(1e-8, 448.0).to(torch.float8_e4m3fn)
    y = v / s.float().clamp_min(2.0 ** -9)[..., None]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    code = torch.bucketize(y.abs(), edges, right=True) + 8 * (y < 0)
    code = code.to(torch.uint8).view(-1, 256, 2)
    return torch.cat([code[..., 0] | (code[..., 1] << 4), s.view(torch.uint8)], 1)


def _lengths(case):
    """(new tokens, context with them) of each sequence: the case's alone, as its work is."""
    r = random.Random(case["mix"])
    new, ctx = [], []
    for b in range(case["batch"]):
        c = case["context"] if b == case["batch"] - 1 else r.randint(max(1, case["context"] // 4), case["context"])
        n = 1 if b < case["decodes"] else case["new"] if b == case["batch"] - 1 else r.randint(max(1, case["new"] // 2), case["new"])
        new.append(min(n, c))
        ctx.append(c)
    return new, ctx


def _requests(case):
    """(slots, tokens before the step, new tokens) of each request: the case's alone."""
    r = random.Random(case["mix"])
    n, fresh = case["requests"], case["context"] == 0
    slots = r.sample(range(case["slots"]), n)
    old = [0 if fresh else r.randint(max(1, case["context"] // 2), case["context"]) for _ in range(n)]
    new = [r.randint(max(1, case["new"] // 2), case["new"]) for _ in range(n)]
    room = case["pages"] // 3                            # no request needs a page that is not there
    for k in range(n):
        old[k] = min(old[k], room // n * case["page"])
        new[k] = min(new[k], max(1, room // n - 1) * case["page"], case["width"] * case["page"] - old[k])
    return slots, old, new


def _live_pages(case, n, c):
    """Pages of a sequence of c tokens, n of them new, that its window still reads."""
    page, width = case["page"], -(-c // case["page"])
    if not case["trim"]:
        return list(range(width))
    lo = max(0, c - n + 1 - case["window"])
    return [j for j in range(width) if j * page < case["sinks"] or (j + 1) * page > lo]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "pages":
        slots, old, new = _requests(case)
        page, S, width, pages = case["page"], case["slots"], case["width"], case["pages"]
        lens = torch.zeros(S, dtype=torch.int64, device="cuda")
        drafts = new if case["kind"] == "spec" else [0] * len(new)      # tokens of the last step, none of them accepted
        lens[torch.tensor(slots, device="cuda")] = torch.tensor([a + b for a, b in zip(old, drafts)], device="cuda")
        need = (lens + page - 1) // page
        perm = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
        at = torch.arange(width, device="cuda")
        tables = torch.where(at < need[:, None], perm[(need.cumsum(0) - need)[:, None] + at.clamp_max(pages - 1 - int(need.sum()))], -1)
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[perm[: int(need.sum())].long()] = 1
        refs[perm[pages - pages // 4:].long()] = 1             # other sequences' pages
        tokens = sum(new) + case["pad"]
        return {"case": case, "tables": tables.int(), "seq": lens.int(), "slots": _ints(slots), "new": _ints(new), "old": _ints(old),
                "refs": refs, "tokens": tokens}
    if op == "rope":
        x = _randn(g, case["tokens"], case["heads"], case["dim"], dtype=DTYPES[case["dtype"]])
        return {"case": case, "x": x, "out": torch.empty_like(x), "pos": _axis_positions(g, case),
                "cos_sin": _cos_sin(case["positions"], case["rotary"]), "axes": _pair_axes(case, case["rotary"])}
    if op == "write":
        T, H, rows = case["tokens"], case["heads"], case["pages"] * case["page"]
        slots = torch.randperm(rows, generator=g, device="cuda")[:T]
        slots[3::11] = -1                                      # padding tokens of a captured batch
        proj = _randn(g, T, H, case["q_dim"])                  # the query projection: its rope part is rotated
        query = torch.zeros(T, H, LATENT + ROPE, dtype=torch.bfloat16, device="cuda")
        return {"case": case, "k_pe": _randn(g, T, LATENT + ROPE)[:, LATENT:], "q_pe": proj[..., case["q_dim"] - ROPE:],
                "query": query, "rope_cache": _randn(g, case["pages"], case["page"], ROPE), "slots": slots,
                "pos": _axis_positions(g, case), "cos_sin": _cos_sin(case["positions"], ROPE), "axes": _pair_axes(case, ROPE)}
    new, ctx = _lengths(case)
    page = case["page"]
    live = [_live_pages(case, n, c) for n, c in zip(new, ctx)]
    pages = sum(len(v) for v in live) + 16
    pool = torch.cat([_pack_nvfp4(_randn(g, min(65536, pages * page - r), LATENT)) for r in range(0, pages * page, 65536)])
    perm = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    tables = torch.full((len(ctx), max(-(-c // page) for c in ctx)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, v in enumerate(live):
        tables[b, torch.tensor(v, device="cuda")] = perm[at: at + len(v)]
        at += len(v)
    cu = _ints([sum(new[:b]) for b in range(len(new) + 1)])
    return {"case": case, "q": _randn(g, sum(new), case["heads"], LATENT + ROPE), "pool": pool.view(pages, page, ROW),
            "rope": _randn(g, pages, page, ROPE) if case["rope"] else None, "tables": tables, "cu": cu, "seq": _ints(ctx),
            "max_new": max(new), "max_ctx": max(ctx)}


# ------------------------------------------------------------------ plain forms
def _drop(refs, ids):
    """One reference less for every id >= 0."""
    refs.index_add_(0, ids.clamp_min(0).flatten().long(), -(ids >= 0).flatten().int())


def _plain_free(s):
    slots = s["slots"].long()
    _drop(s["refs"], s["tables"][slots])
    s["tables"][slots] = -1
    s["seq"][slots] = 0


def _plain_extend(s, old):
    """The requests' tables, and slot, position and sequence of each new token."""
    page, tables, refs, slots = s["case"]["page"], s["tables"], s["refs"], s["slots"].long()
    new, before = s["new"].long(), s["seq"][slots].long()
    at = torch.arange(tables.shape[1], device="cuda")
    end = old + new
    first, last = (old + page - 1) // page, (end + page - 1) // page
    rows = tables[slots]
    kept = (torch.maximum(before, end) + page - 1) // page
    stale = (at >= first[:, None]) & (at < kept[:, None])
    _drop(refs, torch.where(stale, rows, -1))               # pages of tokens that were taken back
    free = torch.argsort((refs != 0).int(), stable=True).int()
    need = last - first
    rank = (need.cumsum(0) - need)[:, None] + at - first[:, None]
    fresh = (at >= first[:, None]) & (at < last[:, None])
    rows = torch.where(fresh, free[rank.clamp(0, free.shape[0] - 1)], torch.where(stale, -1, rows))
    refs.index_add_(0, rows.clamp_min(0).flatten().long(), fresh.flatten().int())
    tables[slots] = rows
    s["seq"][slots] = end.int()
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["tokens"], device="cuda")
    k = torch.searchsorted(cu[1:], t, right=True).clamp_max(new.shape[0] - 1)
    live = t < cu[-1]
    pos = torch.where(live, old[k] + t - cu[k], 0)
    slot = rows[k, pos // page].long() * page + pos % page
    return {"slot_mapping": torch.where(live, slot, -1), "positions": pos.int(), "cu": cu.int(), "lens": end.int(), "batch_tables": rows}


def _plain_trim(s):
    c = s["case"]
    page, slots = c["page"], s["slots"].long()
    rows, lens = s["tables"][slots], s["seq"][slots].long()[:, None]
    first = torch.arange(rows.shape[1], device="cuda") * page
    behind = (rows >= 0) & (first >= c["sinks"]) & (first + page <= lens - c["window"] + 1)
    past = (rows >= 0) & (first >= lens)
    _drop(s["refs"], torch.where(behind | past, rows, -1))
    s["tables"][slots] = torch.where(behind, -2, torch.where(past, -1, rows))


def _plain_pages(s):
    kind = s["case"]["kind"]
    if kind == "window":
        _plain_free(s)
    out = _plain_extend(s, s["seq"][s["slots"].long()].long() if kind == "window" else s["old"].long())
    if kind == "window":
        _plain_trim(s)
    return out


def _rotate(x, c, s, interleaved):
    h = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])
    u, v = a * c - b * s, b * c + a * s
    return torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)


def _angles(s, half):
    """cos and sin of every token's pairs, each pair by its own axis, [tokens, half] each."""
    axes = torch.tensor(s["axes"], device="cuda")
    pos, pair = s["pos"].long()[axes].T, torch.arange(half, device="cuda")
    return s["cos_sin"][pos, pair], s["cos_sin"][pos, half + pair]


def _plain_rope(s):
    c, x = s["case"], s["x"]
    o, r = c["offset"], c["rotary"]
    out = x.clone()
    cos, sin = (v[:, None] for v in _angles(s, r // 2))
    out[..., o:o + r] = _rotate(x[..., o:o + r].float(), cos, -sin if c["inverse"] else sin, c["interleaved"]).to(x.dtype)
    return out


def _plain_write(s):
    c = s["case"]
    cos, sin = _angles(s, ROPE // 2)
    s["query"][..., LATENT:] = _rotate(s["q_pe"].float(), cos[:, None], sin[:, None], c["interleaved"]).to(torch.bfloat16)
    k = _rotate(s["k_pe"].float(), cos, sin, c["interleaved"]).to(torch.bfloat16)
    live = s["slots"] >= 0
    s["rope_cache"].view(-1, ROPE)[s["slots"][live]] = k[live]


def _unpack_nvfp4(rows):
    """288-byte rows -> values, float32."""
    table = torch.tensor(E2M1, device=rows.device)
    code = rows[..., :256].int()
    v = torch.stack([table[code & 15], table[code >> 4]], -1).flatten(-2)
    return v * rows[..., 256:].contiguous().view(torch.float8_e4m3fn).float().repeat_interleave(16, -1)


def _plain_window(s):
    c = s["case"]
    B, H, page, W, S = c["batch"], c["heads"], c["page"], c["window"], c["sinks"]
    Q = s["max_new"]
    cu, seq = s["cu"].long(), s["seq"].long()
    n = cu[1:] - cu[:-1]
    lo = (seq - n + 1 - W).clamp_min(0)[:, None]                                    # the first token in any window
    j = torch.arange(S + min(W + Q - 1, s["max_ctx"]), device="cuda")
    t = torch.where(j < S, j, lo + j - S)                                           # [B, J]
    have = torch.where(j < S, (t < lo) & (t < seq[:, None]), t < seq[:, None])
    t = torch.where(have, t, lo)
    rows = s["tables"].long().gather(1, t // page).clamp_min(0) * page + t % page
    kv = _unpack_nvfp4(s["pool"].view(-1, ROW)[rows])                               # [B, J, 512]
    i = torch.arange(Q, device="cuda")
    at = (cu[:-1, None] + i).clamp_max(max(0, s["q"].shape[0] - 1))                 # [B, Q]
    q = s["q"].float()[at].view(B, Q * H, LATENT + ROPE)
    scores = torch.bmm(q[..., :LATENT], kv.transpose(1, 2))
    if s["rope"] is not None:
        scores += torch.bmm(q[..., LATENT:], s["rope"].view(-1, ROPE)[rows].float().transpose(1, 2))
    own_pos = (seq[:, None] - n[:, None] + i)[..., None]                            # [B, Q, 1]
    t = t[:, None]
    hidden = ~have[:, None] | (t > own_pos) | ((t <= own_pos - W) & (t >= S))
    scores.mul_(SCALE).view(B, Q, H, -1).masked_fill_(hidden[:, :, None], -math.inf)
    top = scores.amax(2, keepdim=True).clamp_min(-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(2, keepdim=True)
    out = torch.bmm(p, kv) / total.clamp_min(1e-30)
    lse = (top + total.log()).view(B, Q, H)
    keep = (i < n[:, None]).flatten().nonzero().flatten()
    return {"out": out.view(B * Q, H, LATENT)[keep].to(torch.bfloat16), "lse": lse.view(B * Q, H)[keep]}


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
    if op == "pages":
        if not own:
            out = _plain_pages(s)
        else:
            window = c["kind"] == "window"
            if window:
                rt.free_pages(s["tables"], s["seq"], s["slots"], s["refs"])
            e = rt.extend_pages(s["tables"], s["seq"], s["slots"], s["new"], s["refs"], c["page"], s["tokens"],
                                lens=None if window else s["old"])
            if window:
                rt.trim_pages(s["tables"], s["seq"], s["slots"], s["refs"], c["page"], window=c["window"], sinks=c["sinks"])
            out = {"slot_mapping": e.slot_mapping, "positions": e.positions, "cu": e.cu_seqlens_q, "lens": e.seq_lens,
                   "batch_tables": e.block_tables}
        return out | {"tables": s["tables"], "seq": s["seq"], "refs": s["refs"]}
    if op == "rope":
        if not own:
            return _plain_rope(s)
        return rt.apply_rope(s["x"], s["pos"], s["cos_sin"], rope_offset=c["offset"], interleaved=c["interleaved"],
                             inverse=c["inverse"], out=s["out"], axes=s["axes"])
    if op == "write":
        if not own:
            _plain_write(s)
        else:
            rt.write_nvfp4_rope_rotated(s["k_pe"], s["rope_cache"], s["slots"], s["pos"], s["cos_sin"], q_pe=s["q_pe"],
                                        q_out=s["query"][..., LATENT:], interleaved=c["interleaved"], axes=s["axes"])
        return {"rope_cache": s["rope_cache"], "query": s["query"]}
    if not own:
        return _plain_window(s)
    out, lse = rt.mla_prefill(s["q"], s["pool"], None, LATENT, ROPE, s["tables"], s["cu"], s["seq"], s["max_new"],
                              s["max_ctx"], bmm1_scale=SCALE, rope_cache=s["rope"], return_lse=True, window=c["window"],
                              sinks=c["sinks"])
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "pages":
        _, old, new = _requests(case)
        n, page = case["requests"], case["page"]
        fresh = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(old, new))
        tokens = sum(new) + case["pad"]
        # the requests, the step's tables read and written, a count and an entry for each new page, 12 bytes a token
        return {"bytes": 20 * n + 8 * n * case["width"] + 16 * fresh + 12 * tokens, "flops": 0}
    if op == "rope":
        size = DTYPES[case["dtype"]].itemsize
        values = case["tokens"] * case["heads"] * case["dim"]
        rot = case["tokens"] * case["heads"] * case["rotary"]
        return {"bytes": 2 * values * size + case["tokens"] * 4 * (case["axes"] + case["rotary"]), "flops": 3 * rot}
    if op == "write":
        T, H = case["tokens"], case["heads"]
        return {"bytes": T * (8 + 4 * case["axes"] + 4 * ROPE + 2 * 2 * ROPE * (H + 1)), "flops": 3 * T * (H + 1) * ROPE}
    new, ctx = _lengths(case)
    H, W, S = case["heads"], case["window"], case["sinks"]
    dims = LATENT + (ROPE if case["rope"] else 0)
    seen = lambda p: min(p + 1, W) + min(S, max(0, p + 1 - W))  # noqa: E731
    pairs = sum(seen(p) for n, c in zip(new, ctx) for p in range(c - n, c))
    rows = 0
    for n, c in zip(new, ctx):
        lo = max(0, c - n + 1 - W)
        rows += c - lo + min(S, lo)
    row = ROW + (2 * ROPE if case["rope"] else 0)
    return {"bytes": rows * row + sum(new) * H * (2 * (dims + LATENT) + 4) + rows // case["page"] * 4,
            "flops": 2 * H * pairs * (dims + LATENT)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None                                            # whole numbers only
    s = prepare(case, seed)
    if op == "window":
        return _exact_window(case, s)
    r = case["rotary"] if op == "rope" else ROPE
    table = torch.complex(s["cos_sin"].double()[:, : r // 2], s["cos_sin"].double()[:, r // 2:])
    T = case["tokens"]
    w = torch.empty(T, r // 2, dtype=torch.complex128, device="cuda")
    for i, a in enumerate(s["axes"]):
        w[:, i] = table[s["pos"][a].long(), i]
    i = torch.arange(r // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
    if op == "rope":
        o = case["offset"]
        out = s["x"].double()
        z = torch.complex(out[..., o + a], out[..., o + b]) * (w.conj() if case["inverse"] else w)[:, None]
        out[..., o + a], out[..., o + b] = z.real, z.imag
        return out
    q, k = s["query"].double(), s["rope_cache"].double().view(-1, ROPE)
    x = s["q_pe"].double()
    z = torch.complex(x[..., a], x[..., b]) * w[:, None]
    q[..., LATENT + a], q[..., LATENT + b] = z.real, z.imag
    x = s["k_pe"].double()
    z = torch.complex(x[..., a], x[..., b]) * w
    y = torch.empty_like(x)
    y[..., a], y[..., b] = z.real, z.imag
    at = s["slots"] >= 0
    k[s["slots"][at]] = y[at]
    return {"rope_cache": k.view(s["rope_cache"].shape), "query": q}


def _exact_window(case, s):
    new, ctx = _lengths(case)
    H, page, W, S, at = case["heads"], case["page"], case["window"], case["sinks"], 0
    grid = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    outs, lses = [], []
    for b, (n, c) in enumerate(zip(new, ctx)):
        lo = max(0, c - n + 1 - W)
        t = torch.tensor([*range(min(S, lo)), *range(lo, c)], device="cuda")
        slot = s["tables"][b].long()[t // page] * page + t % page
        raw = s["pool"].view(-1, ROW)[slot]
        low, high = grid[(raw[:, :256] % 16).long()], grid[(raw[:, :256] // 16).long()]
        kv = torch.stack([low, high], 2).view(-1, 32, 16) * raw[:, 256:].contiguous().view(torch.float8_e4m3fn).double()[..., None]
        kv = kv.view(-1, LATENT)
        q = s["q"][at:at + n].double()
        at += n
        age = (c - n + torch.arange(n, device="cuda"))[:, None] - t[None]
        see = (age >= 0) & ((age < W) | (t < S)[None])
        o = torch.empty(n, H, LATENT, dtype=torch.float64, device="cuda")
        e = torch.empty(n, H, dtype=torch.float64, device="cuda")
        for h in range(H):
            x = q[:, h, :LATENT] @ kv.T
            if s["rope"] is not None:
                x += q[:, h, LATENT:] @ s["rope"].view(-1, ROPE)[slot].double().T
            x = torch.where(see, x * SCALE, -math.inf)
            o[:, h] = torch.softmax(x, 1) @ kv
            e[:, h] = torch.logsumexp(x, 1)
        outs.append(o)
        lses.append(e)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
