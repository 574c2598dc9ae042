"""Serving operators beside the NVFP4 paged cache, as a user calls them, with a plain form of each.

Five operators of one serving step: ``apply_rope`` (rotary positions on queries or keys),
``write_nvfp4_rope_rotated`` (rotated keys into the paged rope side-pool, queries rotated in the
same call), ``mla_prefill`` (attention of a ragged chunk of new tokens over the paged cache) and
the upkeep of the cache's pages, ``free_pages`` + ``fork_pages`` and ``compact_pages``.

With ``own`` false, ``run`` computes them in elementary torch operations in 32 bits; with ``own``
true it makes the framework's calls on the same inputs.
"""
import math
import random

import torch

own = False

LATENT, ROPE, ROW, INDEX_ROW = 512, 64, 288, 72
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 16 sequences: 64 heads of 512 latent + 64 rope dims, latency counts
        {"name": "rope_decode", "op": "rope", "tokens": 16, "heads": 64, "dim": 576, "rotary": 64, "offset": 512,
         "interleaved": True, "inverse": False, "dtype": "bf16", "positions": 131072},
        # the queries of a prefill step, whole heads read and written once
        {"name": "rope_prefill", "op": "rope", "tokens": 8192, "heads": 64, "dim": 576, "rotary": 64, "offset": 512,
         "interleaved": True, "inverse": False, "dtype": "bf16", "positions": 131072},
        # the gradient through the rotation, half layout, an odd token count
        {"name": "rope_backward", "op": "rope", "tokens": 2049, "heads": 32, "dim": 128, "rotary": 64, "offset": 0,
         "interleaved": False, "inverse": True, "dtype": "fp32", "positions": 8192},
        # the write seam of a decode step: 16 tokens, some of them padding
        {"name": "write_decode", "op": "write", "tokens": 16, "heads": 64, "q_dim": 192, "pages": 1024, "page": 64,
         "interleaved": True, "positions": 131072, "dtype": "bf16"},
        # the write seam of 16 chunks of 2048 tokens
        {"name": "write_chunks", "op": "write", "tokens": 32768, "heads": 16, "q_dim": 192, "pages": 4096, "page": 64,
         "interleaved": True, "positions": 300000, "dtype": "bf16"},
        # a speculative step: a few new tokens of each of a few sequences, odd lengths, no rope part
        {"name": "chunk_short", "op": "chunk", "batch": 3, "new": 7, "context": 777, "heads": 16, "page": 64,
         "rope": False, "decodes": 1, "mix": 5},
        # single tokens of a batch of 16 with contexts up to 8K
        {"name": "chunk_single", "op": "chunk", "batch": 16, "new": 1, "context": 8192, "heads": 64, "page": 64,
         "rope": True, "decodes": 16, "mix": 3},
        # a mixed serving step: two chunks among single-token sequences
        {"name": "chunk_mixed", "op": "chunk", "batch": 8, "new": 777, "context": 8192, "heads": 32, "page": 64,
         "rope": True, "decodes": 6, "mix": 4},
        # a 2048-token chunk of a long prompt, 64 heads: compute-bound
        {"name": "chunk_prefill", "op": "chunk", "batch": 1, "new": 2048, "context": 16384, "heads": 64, "page": 64,
         "rope": True, "decodes": 0, "mix": 2},
        # a beam step: the old beams' pages are freed and the surviving ones forked
        {"name": "fork_beams", "op": "fork", "parents": 4, "children": 28, "context": 2000, "pages": 1024, "page": 64,
         "mix": 1},
        # many samples of long prompts in a pool of about 2.7 million tokens
        {"name": "fork_samples", "op": "fork", "parents": 32, "children": 480, "context": 16000, "pages": 42405,
         "page": 64, "mix": 7},
        # the same pool after half of its sequences ended: live pages move to its front
        {"name": "compact_pool", "op": "compact", "slots": 256, "context": 8192, "pages": 42405, "page": 64,
         "live": 0.6, "mix": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "chunk", "chunk", "fork", "compact"])
    if op == "rope":
        rotary = rng.choice([16, 32, 64, 128])
        dim, offset = rng.choice([(576, 576 - rotary), (128, 0), (192, 192 - rotary)])
        heads = rng.randint(1, 64)
        return {"op": op, "tokens": _log(rng, 1, 8192 * 64 * 576 // (4 * heads * dim)), "heads": heads, "dim": dim,
                "rotary": min(rotary, dim), "offset": offset, "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.3, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "positions": rng.choice([8192, 131072])}
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 30000), "heads": rng.randint(1, 32), "q_dim": rng.choice([64, 192]),
                "pages": rng.randint(1000, 2000) * 64 // 16, "page": rng.choice([16, 64]),
                "interleaved": rng.random() < 0.5, "positions": rng.choice([8192, 131072]), "dtype": "bf16"}
    if op == "chunk":
        context = _log(rng, 1, 16384)
        batch = rng.randint(1, 8)
        heads = rng.choice([1, 4, 16, 20, 32, 64, 128])
        new = _log(rng, 1, max(1, min(context, 1500000000 // (batch * heads * context))))
        return {"op": op, "batch": batch, "new": new, "context": context, "heads": heads,
                "page": rng.choice([16, 64, 128]), "rope": rng.random() < 0.7, "decodes": rng.randint(0, batch),
                "mix": rng.randint(0, 1 << 20)}
    if op == "fork":
        parents = rng.randint(1, 24)
        context = _log(rng, 64, 8000)
        children = _log(rng, 1, 400)
        page = rng.choice([16, 64])
        need = parents * (context // page + 1) + children
        return {"op": op, "parents": parents, "children": children, "context": context,
                "pages": need + rng.randint(64, 4096), "page": page, "mix": rng.randint(0, 1 << 20)}
    pages = _log(rng, 300, 40000)
    return {"op": op, "slots": rng.randint(2, 128), "context": _log(rng, 64, 4096), "pages": pages, "page": 64,
            "live": rng.uniform(0.2, 0.9), "mix": rng.randint(0, 1 << 20)}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _cos_sin(positions, rotary, factor=4.0):
    """cos | sin of every position, [positions, rotary] float32: long contexts by scaled frequencies."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary) / factor
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


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


def _caches(g, pages, page):
    """The three pools of a cache: latent rows, rope rows, indexer rows."""
    b = lambda w: torch.randint(0, 256, (pages, page, w), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    return [b(ROW), _randn(g, pages, page, ROPE), b(INDEX_ROW)]


def _sequences(g, slots, lens, pages, page):
    """Page tables of `slots` sequences with pages drawn at random, -1 padded, and reference counts."""
    width = max(1, max(-(-n // page) for n in lens))
    need = [-(-n // page) for n in lens]
    perm = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    at = torch.arange(width, device="cuda")
    n = torch.tensor(need, device="cuda")
    start = n.cumsum(0) - n
    t = perm[(start[:, None] + at).clamp_max(pages - 1)]
    tables = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
    tables[: len(lens)] = torch.where(at < n[:, None], t, -1)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[perm[: sum(need)].long()] = 1
    seq = torch.zeros(slots, dtype=torch.int32, device="cuda")
    seq[: len(lens)] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return tables, refs, seq


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "rope":
        x = _randn(g, case["tokens"], case["heads"], case["dim"], dtype=DTYPES[case["dtype"]])
        return {"case": case, "x": x, "out": torch.empty_like(x),
                "pos": torch.randint(0, case["positions"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32),
                "cos_sin": _cos_sin(case["positions"], case["rotary"])}
    if op == "write":
        T, H, rows = case["tokens"], case["heads"], case["pages"] * case["page"]
        slots = torch.randperm(rows, generator=g, device="cuda")[:T]
        slots[3::11] = -1                                      # padding tokens of a captured batch
        proj = _randn(g, T, H, case["q_dim"])                  # the query projection: its rope part is rotated
        query = torch.zeros(T, H, LATENT + ROPE, dtype=torch.bfloat16, device="cuda")
        return {"case": case, "k_pe": _randn(g, T, LATENT + ROPE)[:, LATENT:], "q_pe": proj[..., case["q_dim"] - ROPE:],
                "query": query, "rope_cache": _randn(g, case["pages"], case["page"], ROPE), "slots": slots,
                "pos": torch.randint(0, case["positions"], (T,), generator=g, device="cuda", dtype=torch.int32),
                "cos_sin": _cos_sin(case["positions"], ROPE)}
    if op == "chunk":
        new, ctx = _lengths(case)
        page, need = case["page"], sum(-(-c // case["page"]) for c in ctx)
        pages = need + 16
        pool = torch.cat([_pack_nvfp4(_randn(g, min(65536, pages * page - r), LATENT)) for r in range(0, pages * page, 65536)])
        tables, _, _ = _sequences(g, len(ctx), ctx, pages, page)
        cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        return {"case": case, "q": _randn(g, sum(new), case["heads"], LATENT + ROPE), "pool": pool.view(pages, page, ROW),
                "rope": _randn(g, pages, page, ROPE) if case["rope"] else None, "tables": tables, "cu": cu,
                "seq": torch.tensor(ctx, dtype=torch.int32, device="cuda"), "max_new": max(new), "max_ctx": max(ctx)}
    r = random.Random(case["mix"])
    if op == "fork":
        P, C = case["parents"], case["children"]
        lens = [r.randint(max(1, case["context"] // 2), case["context"]) for _ in range(P)]
        caches = _caches(g, case["pages"], case["page"])
        tables, refs, seq = _sequences(g, P + C, lens, case["pages"], case["page"])
        src = torch.randint(0, P, (C,), generator=g, device="cuda", dtype=torch.int32)
        dst = P + torch.randperm(C, generator=g, device="cuda", dtype=torch.int32)
        s = {"case": case, "caches": caches, "tables": tables, "refs": refs, "seq": seq, "src": src, "dst": dst}
        _fork(s)                                               # the beams of the step before
        return s
    budget = int(case["pages"] * case["live"])
    lens, used = [], 0
    for _ in range(case["slots"]):
        n = r.randint(1, case["context"])
        n = min(n, (budget - used) * case["page"])
        lens.append(n)
        used += -(-n // case["page"])
    caches = _caches(g, case["pages"], case["page"])
    tables, refs, _ = _sequences(g, case["slots"], lens, case["pages"], case["page"])
    refs += (refs > 0).int() * torch.randint(0, 3, refs.shape, generator=g, device="cuda", dtype=torch.int32)
    return {"case": case, "caches": caches, "tables": tables, "refs": refs, "out_tables": torch.empty_like(tables),
            "out_refs": torch.empty_like(refs)}


# ------------------------------------------------------------------ plain forms
def _rotate(x, cs, interleaved, inverse=False):
    """The rotation of x [..., r] by cs [..., r] = cos | sin, in x's precision."""
    h = x.shape[-1] // 2
    c, s = cs[..., :h], cs[..., h:]
    s = -s if inverse else s
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])
    u, v = a * c - b * s, b * c + a * s
    return torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)


def _plain_rope(s):
    c, x = s["case"], s["x"]
    o, r = c["offset"], c["rotary"]
    out = x.clone()
    cs = s["cos_sin"][s["pos"].long()][:, None]
    out[..., o:o + r] = _rotate(x[..., o:o + r].float(), cs, c["interleaved"], c["inverse"]).to(x.dtype)
    return out


def _plain_write(s):
    c = s["case"]
    cs = s["cos_sin"][s["pos"].long()]
    s["query"][..., LATENT:] = _rotate(s["q_pe"].float(), cs[:, None], c["interleaved"]).to(torch.bfloat16)
    k = _rotate(s["k_pe"].float(), cs, c["interleaved"]).to(torch.bfloat16)
    rows = s["rope_cache"].view(-1, ROPE)
    live = s["slots"] >= 0
    rows[s["slots"][live]] = k[live]


def _unpack_nvfp4(rows):
    """288-byte rows -> values, float32."""
    table = torch.tensor(E2M1, device=rows.device)
    code = rows[..., :256].int()
    v = torch.stack([table[code & 15], table[code >> 4]], -1).flatten(-2)
    return v * rows[..., 256:].contiguous().view(torch.float8_e4m3fn).float().repeat_interleave(16, -1)


def _plain_chunk(s):
    c = s["case"]
    B, H, page, Q, L = c["batch"], c["heads"], c["page"], s["max_new"], s["max_ctx"]
    t = torch.arange(L, device="cuda")
    rows = s["tables"][:, t // page].long() * page + t % page                       # [B, L]
    rows = rows.clamp_min(0)
    kv = _unpack_nvfp4(s["pool"].view(-1, ROW)[rows])                               # [B, L, 512]
    cu, seq = s["cu"].long(), s["seq"].long()
    n = cu[1:] - cu[:-1]
    i = torch.arange(Q, device="cuda")
    at = (cu[:-1, None] + i).clamp_max(max(0, s["q"].shape[0] - 1))                 # [B, Q]
    q = s["q"].float()[at].view(B, Q * H, LATENT + ROPE)
    scores = torch.bmm(q[..., :LATENT], kv.transpose(1, 2))
    if s["rope"] is not None:
        k_pe = s["rope"].view(-1, ROPE)[rows].float()
        scores += torch.bmm(q[..., LATENT:], k_pe.transpose(1, 2))
    limit = seq[:, None] - n[:, None] + i + 1                                       # tokens each query sees
    hidden = (t >= limit[..., None])[:, :, None].expand(B, Q, H, L).reshape(B, Q * H, L)
    scores = scores.mul_(SCALE).masked_fill_(hidden, -math.inf)
    top = scores.amax(2, keepdim=True).clamp_min(-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(2, keepdim=True)
    out = torch.bmm(p, kv) / total.clamp_min(1e-30)
    lse = (top + total.log()).view(B, Q, H)
    keep = (i < n[:, None]).flatten().nonzero().flatten()
    return {"out": out.view(B * Q, H, LATENT)[keep].to(torch.bfloat16), "lse": lse.view(B * Q, H)[keep]}


SCALE = 1.0 / 24.0


def _free(s):
    """The children's pages go back: one reference less each, their tables emptied."""
    slots = s["dst"].long()
    ids = s["tables"][slots]
    s["refs"].index_add_(0, ids.clamp_min(0).flatten().long(), -(ids >= 0).flatten().int()).clamp_min_(0)
    s["tables"][slots] = -1
    s["seq"][slots] = 0


def _fork(s):
    """Each child shares its parent's full pages and gets a copy of the last one, in the lowest free page."""
    page, tables, refs = s["case"]["page"], s["tables"], s["refs"]
    src, dst = s["src"].long(), s["dst"].long()
    ids, lens = tables[src], s["seq"][src]
    full, rest = lens // page, lens % page
    at = torch.arange(tables.shape[1], device=tables.device)
    need = rest > 0
    free = torch.argsort((refs != 0).int(), stable=True)
    rank = (need.int().cumsum(0) - 1).clamp_min(0)
    fresh = free[rank.long()].int()
    shared = at < full[:, None]
    refs.index_add_(0, ids.clamp_min(0).flatten().long(), shared.flatten().int())
    old = ids.gather(1, full.long().clamp_max(tables.shape[1] - 1)[:, None])[:, 0].clamp_min(0)
    old = torch.where(need, old, ids[:, 0])
    to = torch.where(need, fresh, old).long()
    refs.index_add_(0, to, need.int())
    row = torch.arange(page, device=tables.device)
    move = (row < rest[:, None])[..., None]
    for pool in s["caches"]:
        pool[to] = torch.where(move, pool[old.long()], pool[to])
    last = (at == full[:, None]) & need[:, None]
    tables[dst] = torch.where(shared, ids, torch.where(last, fresh[:, None], -1))
    s["seq"][dst] = lens


def _plain_compact(s):
    """The pages in use move to the front of the pools: the k-th one past the front into its k-th hole."""
    refs, tables = s["refs"], s["tables"]
    idx = torch.arange(refs.shape[0], device=refs.device)
    live = refs > 0
    n = live.sum()
    src, dst = (live & (idx >= n)).nonzero().flatten(), (~live & (idx < n)).nonzero().flatten()
    remap = idx.int()
    remap[src] = dst.int()
    for pool in s["caches"]:
        pool[dst] = pool[src]
    s["out_tables"].copy_(torch.where(tables >= 0, remap[tables.clamp_min(0).long()], -1))
    out = refs.clone()
    out[dst] = refs[src]
    out[src] = 0
    s["out_refs"].copy_(out)
    return n.int()


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
    if op == "rope":
        if not own:
            return _plain_rope(s)
        return rt.apply_rope(s["x"], s["pos"], s["cos_sin"], rope_offset=c["offset"], interleaved=c["interleaved"],
                             inverse=c["inverse"], out=s["out"])
    if op == "write":
        if not own:
            _plain_write(s)
        else:
            rt.write_nvfp4_rope_rotated(s["k_pe"], s["rope_cache"], s["slots"], s["pos"], s["cos_sin"], q_pe=s["q_pe"],
                                        q_out=s["query"][..., LATENT:], interleaved=c["interleaved"])
        return {"rope_cache": s["rope_cache"], "query": s["query"]}
    if op == "chunk":
        if not own:
            return _plain_chunk(s)
        out, lse = rt.mla_prefill(s["q"], s["pool"], None, LATENT, ROPE, s["tables"], s["cu"], s["seq"], s["max_new"],
                                  s["max_ctx"], bmm1_scale=SCALE, rope_cache=s["rope"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "fork":
        if not own:
            _free(s)
            _fork(s)
        else:
            rt.free_pages(s["tables"], s["seq"], s["dst"], s["refs"])
            rt.fork_pages(s["caches"], s["tables"], s["seq"], s["src"], s["dst"], s["refs"])
        return {"tables": s["tables"], "seq": s["seq"], "refs": s["refs"], "caches": s["caches"]}
    if not own:
        n = _plain_compact(s)
    else:
        n = rt.compact_pages(s["caches"], s["tables"], s["refs"], out_tables=s["out_tables"], out_ref_counts=s["out_refs"])
    return {"live": n, "tables": s["out_tables"], "refs": s["out_refs"], "caches": s["caches"]}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "rope":
        size = DTYPES[case["dtype"]].itemsize
        values = case["tokens"] * case["heads"] * case["dim"]
        rot = case["tokens"] * case["heads"] * case["rotary"]
        return {"bytes": 2 * values * size + case["tokens"] * (4 + 4 * case["rotary"]), "flops": 3 * rot}
    if op == "write":
        T, H = case["tokens"], case["heads"]
        return {"bytes": T * (8 + 4 + 4 * ROPE + 2 * 2 * ROPE * (H + 1)), "flops": 3 * T * (H + 1) * ROPE}
    if op == "chunk":
        new, ctx = _lengths(case)
        H = case["heads"]
        dims = LATENT + (ROPE if case["rope"] else 0)
        pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, ctx))
        row = ROW + (2 * ROPE if case["rope"] else 0)
        return {"bytes": sum(ctx) * row + sum(new) * H * 2 * (dims + LATENT + 2) + sum(ctx) // case["page"] * 4,
                "flops": 2 * H * pairs * (dims + LATENT)}
    page_bytes = case["page"] * (ROW + 2 * ROPE + INDEX_ROW)
    if op == "fork":
        r = random.Random(case["mix"])
        lens = [r.randint(max(1, case["context"] // 2), case["context"]) for _ in range(case["parents"])]
        width = max(-(-n // case["page"]) for n in lens)
        # the children's tables read, written and emptied, a count up and down for each, half a page copied
        return {"bytes": case["children"] * (4 * width * 4 + page_bytes) + 4 * case["pages"], "flops": 0}
    used = min(int(case["pages"] * case["live"]), case["slots"] * (case["context"] // case["page"]) // 2)
    moved = used * (case["pages"] - used) // case["pages"]
    return {"bytes": 2 * moved * page_bytes + 8 * case["pages"] + 8 * used, "flops": 0}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None                                            # whole numbers and copied bytes only
    s = prepare(case, seed)
    if op == "rope":
        c, r, o = case, case["rotary"], case["offset"]
        cs = s["cos_sin"].double()[s["pos"].long()]
        w = torch.complex(cs[:, None, : r // 2], -cs[:, None, r // 2:] if c["inverse"] else cs[:, None, r // 2:])
        out = s["x"].double()
        part = out[..., o:o + r]
        i = torch.arange(r // 2, device="cuda")
        a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + r // 2)
        z = torch.complex(part[..., a], part[..., b]) * w
        part[..., a], part[..., b] = z.real, z.imag
        return out
    if op == "write":
        cs = s["cos_sin"].double()[s["pos"].long()]
        w = torch.complex(cs[:, : ROPE // 2], cs[:, ROPE // 2:])
        i = torch.arange(ROPE // 2, device="cuda")
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + ROPE // 2)
        q, k = s["query"].double(), s["rope_cache"].double().view(-1, ROPE)
        x = s["q_pe"].double()
        z = torch.complex(x[..., a], x[..., b]) * w[:, None]
        q[..., LATENT + a], q[..., LATENT + b] = z.real, z.imag
        x = s["k_pe"].double()
        z = torch.complex(x[..., a], x[..., b]) * w
        y = torch.empty_like(x)
        y[..., a], y[..., b] = z.real, z.imag
        for t, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                k[slot] = y[t]
        return {"rope_cache": k.view(s["rope_cache"].shape), "query": q}
    new, ctx = _lengths(case)
    H, page, at = case["heads"], case["page"], 0
    grid = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    outs, lses = [], []
    for b, (n, c) in enumerate(zip(new, ctx)):
        t = torch.arange(c, device="cuda")
        slot = s["tables"][b].long()[t // page] * page + t % page
        raw = s["pool"].view(-1, ROW)[slot]
        lo, hi = grid[(raw[:, :256] % 16).long()], grid[(raw[:, :256] // 16).long()]
        kv = torch.stack([lo, hi], 2).view(c, 32, 16) * raw[:, 256:].contiguous().view(torch.float8_e4m3fn).double()[..., None]
        kv = kv.view(c, LATENT)
        q = s["q"][at:at + n].double()
        at += n
        see = t[None] <= (c - n + torch.arange(n, device="cuda"))[:, None]
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
