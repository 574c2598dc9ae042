"""GPU: chunk attention over long contexts (131,072 tokens and more), row by row against the formula in
64 bits.

Tolerance of an output element y = sum_t p_t v_t: one rounding to bf16 (2^-8 |y|), the probabilities'
rounding to 11 bits and the scores' fp32 accumulation, as over short contexts ((2^-11 + 2 dS) A,
A = sum_t p_t |v_t|), the sum of the row in fp32 (its 64 partial sums of a tile's quarter each add
L / 256 values, 2^-24 of the running sum each: L 2^-32 A), the output's fp32 accumulation in the tensor
core, 16 tokens at a time (L / 16 additions that may each cut 2^-23 of the running sum: L 2^-27 A), and
what fp16 cannot hold of small probabilities: they are kept relative to 2^7 at the largest, so that a
rounding below fp16's smallest normal number is at most 2^-25 / 2^7 = 2^-32 of it (2^-32 sum_t |v_t|)."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_gpu import GRID

pytestmark = pytest.mark.gpu
PAGE = 64


def latents(rows):
    """288-byte rows -> float64 values, on the GPU."""
    grid = GRID.to(rows.device)
    v = torch.stack([grid[(rows[:, :256] & 15).long()], grid[(rows[:, :256] >> 4).long()]], 2).view(-1, 32, 16)
    return (v * rows[:, 256:].contiguous().view(torch.float8_e4m3fn).double()[..., None]).view(-1, 512)


class Long:
    """Sequences over a pool of random rows; `spread` scales the latents, `shift` is added to each."""

    def __init__(self, new, ctx, H, seed, spread=1.0, shift=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.new, self.ctx, self.H, self.scale = new, ctx, H, 1.0 / 24.0
        need = [-(-c // PAGE) for c in ctx]
        self.pages = sum(need) + 5
        self.pool = torch.empty(self.pages, PAGE, 288, dtype=torch.uint8, device="cuda")
        for r in range(0, self.pages * PAGE, 1 << 18):
            n = min(1 << 18, self.pages * PAGE - r)
            x = spread * torch.randn(n, 512, generator=g, device="cuda")
            rt.write_nvfp4((x if shift is None else x + shift).to(torch.bfloat16), self.pool, torch.arange(r, r + n, device="cuda"))
        self.rope = torch.randn(self.pages, PAGE, 64, generator=g, device="cuda").to(torch.bfloat16)
        perm = torch.randperm(self.pages, generator=g, device="cuda").int()
        self.tables = torch.full((len(ctx), max(need)), -1, dtype=torch.int32, device="cuda")
        for b, n in enumerate(need):
            self.tables[b, :n] = perm[sum(need[:b]):sum(need[:b]) + n]
        self.q = torch.randn(sum(new), H, 576, generator=g, device="cuda").to(torch.bfloat16)

    def slots(self, b):
        t = torch.arange(self.ctx[b], device="cuda")
        return self.tables[b].long()[t // PAGE] * PAGE + t % PAGE

    def run(self):
        cu = torch.tensor([sum(self.new[:b]) for b in range(len(self.new) + 1)], dtype=torch.int32, device="cuda")
        return rt.mla_prefill(self.q, self.pool, None, 512, 64, self.tables, cu, torch.tensor(self.ctx, dtype=torch.int32, device="cuda"),
                              max(self.new), max(self.ctx), bmm1_scale=self.scale, rope_cache=self.rope, return_lse=True)

    def check(self, out, lse, rows=None):
        """Every row, or the (token, head) rows of each sequence that `rows` names."""
        at = 0
        for b, (n, c) in enumerate(zip(self.new, self.ctx)):
            slot = self.slots(b)
            v = latents(self.pool.view(-1, 288)[slot])
            k = torch.cat([v, self.rope.view(-1, 64)[slot].double()], 1)
            i, h = torch.tensor(rows or [(i, h) for i in range(n) for h in range(self.H)], device="cuda").T
            q = self.q[at + i, h].double()
            see = torch.arange(c, device="cuda")[None] <= (c - n + i)[:, None]
            x = torch.where(see, (q @ k.T) * self.scale, -torch.inf)
            e = torch.logsumexp(x, 1)
            p = (x - e[:, None]).exp()
            top = x.amax(1)
            y, A = p @ v, p @ v.abs()
            dS = 576 * 2.0 ** -24 * self.scale * (q.abs() @ k.abs().T).amax(1)
            lost = 2.0 ** -32 * (see.double() @ v.abs()) * (top - e).exp()[:, None]
            tol = 2.0 ** -8 * y.abs() + (2.0 ** -11 + 2 * dS + c * (2.0 ** -27 + 2.0 ** -32))[:, None] * A + lost
            got = out[at + i, h].double()
            assert bool(((got - y).abs() <= tol).all()), (b, float((got - y).abs().max()), float(((got - y).abs() / tol).max()))
            err = (lse[at + i, h].double() - e).abs()
            assert bool((err <= dS + 2.0 ** -20 + c * 2.0 ** -32 + 2.0 ** -22 * e.abs()).all()), (b, float(err.max()))
            at += n


@pytest.mark.parametrize("new,ctx,H", [([1], [131072], 4), ([2], [131073], 64), ([1, 5, 64], [200001, 131072, 300000], 3)])
def test_long_contexts(new, ctx, H):
    p = Long(new, ctx, H, seed=H)
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)


def test_chunk_over_a_long_context():
    p = Long([2048], [300000], 8, seed=1)
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse, rows=[(0, 0), (1, 7), (777, 3), (1023, 5), (1024, 0), (2046, 6), (2047, 7)])


def test_real_images_of_more_than_the_cap_run_in_groups():
    """Nine contexts whose images take 1.3 GB: the batch runs in two groups."""
    p = Long([1, 3, 1, 1, 2, 1, 1, 1, 4], [131072] * 8 + [100001], 3, seed=2)
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)


@pytest.mark.parametrize("below", [15.0, 18.0, 20.0])
@pytest.mark.parametrize("new,H,sink", [(1, 2, 0), (1, 2, 131070), (2048, 8, 0), (2048, 8, 77777)])
def test_a_sink_over_a_long_flat_tail(new, H, sink, below):
    """One token with a value of zero takes nearly all of the weight; the output is what the others,
    exp(-below) of it each, add up to.  A single token's work is cut into parts with a maximum of their
    own; the rows of a long chunk meet the sink and the tail in one."""
    shift = torch.randn(512, generator=torch.Generator().manual_seed(5)).cuda()
    p = Long([new], [131072], H, seed=6, spread=0.3, shift=shift)
    p.q[..., :512] *= 0.02
    rope = p.rope.view(-1, 64)
    rope[:] = 0
    slot = p.slots(0)[sink]
    p.pool.view(-1, 288)[slot] = 0
    p.q[..., 512:] = 1.0
    rope[slot] = below * 24.0 / 64.0
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse, rows=None if new == 1 else [(0, 0), (1, 7), (777, 3), (1024, 5), (2047, 6)])
    assert float(out.float().abs().max()) > 0.0
