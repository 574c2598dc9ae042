"""A small serving loop over the NVFP4 paged cache, as an engine would use the operators together:

    python -m glm53_flash_dual_dgx_spark_b200.serving_step [--heads 64] [--prompt 700] [--steps 3]

Two prompts are prefilled in chunks (latents appended, keys and queries rotated, attention of the
chunk over everything cached), one of them is forked into samples that decode on, the samples
end, and the pool is compacted.  Random weights stand in for the model: what it shows is the
order of the calls and that the cache survives them (the attention of a sequence is the same
before and after its pages move, and a fork's first step equals its parent's).
"""
from __future__ import annotations

import argparse

import torch

from . import glm53_nvfp4_runtime as rt

PAGE = 64


class Cache:
    """The pools of one layer, and the tables of the sequences that live in them."""

    def __init__(self, num_pages: int, slots: int, max_tokens: int, device):
        self.latent = torch.zeros(num_pages, PAGE, rt.NV_BYTES, dtype=torch.uint8, device=device)
        self.rope = torch.zeros(num_pages, PAGE, rt.ROPE, dtype=torch.bfloat16, device=device)
        self.tables = torch.full((slots, -(-max_tokens // PAGE)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device=device)

    @property
    def pools(self):
        return [self.latent, self.rope]

    def extend(self, slot: int, n: int) -> torch.Tensor:
        """Pages for n more tokens of a sequence (a host-side scheduler's choice); their pool slots."""
        have = int(self.lens[slot])
        free = (self.refs == 0).nonzero().flatten()
        first, last = -(-have // PAGE), -(-(have + n) // PAGE)
        pages = free[: last - first].int()
        if pages.numel() < last - first:
            raise RuntimeError("the cache is full")
        self.tables[slot, first:last] = pages
        self.refs[pages.long()] = 1
        self.lens[slot] = have + n
        t = torch.arange(have, have + n, device=self.lens.device)
        return self.tables[slot, t // PAGE].long() * PAGE + t % PAGE


def attend(cache: Cache, slots, q, new, cos_sin, positions, write_slots, kv_c, k_pe, scale):
    """One layer's step for the new tokens of `slots`: append, rotate, attend."""
    rt.write_nvfp4(kv_c, cache.latent, write_slots)
    rt.write_nvfp4_rope_rotated(k_pe, cache.rope, write_slots, positions, cos_sin, q_pe=q[..., rt.LATENT:])
    return read(cache, slots, q, new, scale)


def read(cache: Cache, slots, q, new, scale):
    rows = torch.tensor(slots, device=q.device)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=q.device)
    return rt.mla_prefill(q, cache.latent, None, rt.LATENT, rt.ROPE, cache.tables[rows], cu, cache.lens[rows],
                          max(new), cache.tables.shape[1] * PAGE, bmm1_scale=scale, rope_cache=cache.rope)


def run(heads: int = 64, prompt: int = 700, steps: int = 3, chunk: int = 256, seed: int = 0, device="cuda") -> dict:
    g = torch.Generator(device=device).manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=g, device=device).to(torch.bfloat16)  # noqa: E731
    lens, samples = [prompt, prompt // 2], 4
    max_tokens = prompt + steps
    cache = Cache(4 * -(-max_tokens // PAGE) + samples + 8, 2 + samples, max_tokens, device)
    cos_sin = rt.rope_cos_sin(max(max_tokens, 4096), factor=4.0, original_positions=1024, device=device)
    scale = (rt.LATENT + rt.ROPE) ** -0.5

    def step(slots, new):
        first = [int(cache.lens[s]) for s in slots]
        write = torch.cat([cache.extend(s, n) for s, n in zip(slots, new)])
        positions = torch.cat([torch.arange(f, f + n, device=device) for f, n in zip(first, new)])
        T = sum(new)
        q, kv, kr = draw(T, heads, rt.LATENT + rt.ROPE), draw(T, rt.LATENT), draw(T, rt.ROPE)
        return attend(cache, slots, q, new, cos_sin, positions, write, kv, kr, scale), q

    # chunked prefill of both prompts
    done = [0, 0]
    while done != lens:
        new = [min(chunk, n - d) for n, d in zip(lens, done)]
        slots = [s for s, n in enumerate(new) if n]
        out, q = step(slots, [n for n in new if n])
        done = [d + n for d, n in zip(done, new)]
    # samples of the first prompt: full pages shared, the last one copied
    src = torch.zeros(samples, dtype=torch.int32, device=device)
    dst = torch.arange(2, 2 + samples, dtype=torch.int32, device=device)
    probe = draw(1, heads, rt.LATENT + rt.ROPE)
    parent = read(cache, [0], probe, [1], scale)
    rt.fork_pages(cache.pools, cache.tables, cache.lens, src, dst, cache.refs)
    forked = read(cache, [2 + samples - 1], probe, [1], scale)
    shared = int((cache.refs > 1).sum())
    for _ in range(steps):                      # every sequence decodes a token
        step(list(range(2 + samples)), [1] * (2 + samples))
    # the second prompt and two samples end; the rest moves to the front of the pool
    before = read(cache, [0, 2], torch.cat([probe, probe]), [1, 1], scale)
    rt.free_pages(cache.tables, cache.lens, torch.tensor([1, 3, 4], dtype=torch.int32, device=device), cache.refs)
    live = rt.compact_pages(cache.pools, cache.tables, cache.refs)
    after = read(cache, [0, 2], torch.cat([probe, probe]), [1, 1], scale)
    return {"fork_equals_parent": bool(torch.equal(parent, forked)), "compaction_keeps_outputs": bool(torch.equal(before, after)),
            "shared_pages": shared, "live_pages": int(live), "highest_page": int(cache.tables.max()),
            "device_errors": rt.device_errors(), "out": out}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--heads", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--steps", type=int, default=3)
    a = ap.parse_args()
    got = run(a.heads, a.prompt, a.steps)
    del got["out"]
    print(got)


if __name__ == "__main__":
    main()
