"""GPU: causal MLA attention of ragged chunks over the NVFP4 paged pool against the formula in 64
bits.

Tolerance of an output element y = sum_t p_t v_t: one rounding to bf16 (2^-8 |y|), the
probabilities' rounding to 11 bits (2^-11 A, A = sum_t p_t |v_t|), and the scores' fp32
accumulation over 576 products, dS = 576 * 2^-24 * max_t |scale| sum_d |q_d k_d|, which moves
each p by a factor of at most e^dS and their sum by as much (2 dS A); probabilities too small
for fp16 lose at most 2^-25 each (2^-25 sum_t |v_t|).  lse moves by at most dS plus the fp32
rounding of itself and of the exponentials (2^-20)."""
import math

import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt

pytestmark = pytest.mark.gpu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                    dtype=torch.float64)


def latents(rows):
    """288-byte rows -> float64 values (NaN scales stay NaN)."""
    rows = rows.cpu()
    v = torch.stack([GRID[(rows[:, :256] & 15).long()], GRID[(rows[:, :256] >> 4).long()]], 2).view(-1, 32, 16)
    return (v * rows[:, 256:].contiguous().view(torch.float8_e4m3fn).double()[..., None]).view(-1, 512)


class Problem:
    def __init__(self, new, ctx, H, page=64, rope=True, seed=0, spare=3, q_gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.ctx, self.H, self.page = new, ctx, H, page
        need = [-(-c // page) for c in ctx]
        self.pages = sum(need) + spare
        self.width = max(1, max(need))
        x = torch.randn(self.pages * page, 512, generator=g)
        x[::37] *= 4.0
        self.pool = torch.zeros(self.pages, page, 288, dtype=torch.uint8, device="cuda")
        rt.write_nvfp4(x.to(torch.bfloat16).cuda(), self.pool, torch.arange(self.pages * page, device="cuda"))
        self.rope = torch.randn(self.pages, page, 64, generator=g).to(torch.bfloat16).cuda() if rope else None
        perm = torch.randperm(self.pages, generator=g).tolist()
        self.tables = torch.full((len(ctx), self.width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            self.tables[b, :n] = torch.tensor([perm.pop() for _ in range(n)], dtype=torch.int32)
        self.q = (q_gain * torch.randn(sum(new), H, 576, generator=g)).to(torch.bfloat16).cuda()
        self.scale = 1.0 / 24.0

    def slots(self, b):
        t = torch.arange(self.ctx[b])
        p = self.tables[b].long()[t // self.page]
        return torch.where((p >= 0) & (p < self.pages), p * self.page + t % self.page, -1)

    def run(self, **kw):
        cu = torch.tensor([sum(self.new[:b]) for b in range(len(self.new) + 1)], dtype=torch.int32, device="cuda")
        seq = torch.tensor(self.ctx, dtype=torch.int32, device="cuda")
        args = dict(bmm1_scale=self.scale, rope_cache=self.rope, return_lse=True) | kw
        return rt.mla_prefill(args.pop("q", self.q), self.pool, None, 512, 64, self.tables.cuda(), cu, seq,
                              max(self.new), max(self.ctx), **args)

    def check(self, out, lse, out_scale=1.0):
        at = 0
        for b, (n, c) in enumerate(zip(self.new, self.ctx)):
            slot = self.slots(b)
            kv = latents(self.pool.view(-1, 288).cpu()[slot.clamp_min(0)])
            kr = self.rope.view(-1, 64).cpu()[slot.clamp_min(0)].double() if self.rope is not None else None
            q = self.q[at:at + n].cpu().double().reshape(n * self.H, 576)
            k = kv if kr is None else torch.cat([kv, kr], 1)
            q = q[:, : k.shape[1]]
            i = torch.arange(n).repeat_interleave(self.H)
            see = (torch.arange(c)[None] <= (c - n + i)[:, None]) & (slot >= 0)[None]
            kz = torch.nan_to_num(k, nan=0.0)
            x = torch.where(see, (q @ kz.T) * self.scale, -math.inf)
            bad = torch.isnan(k).any(1)                     # a token whose latent holds a NaN
            poisoned = (see & bad[None]).any(1)
            seen = see.any(1)
            top = torch.where(seen, x.amax(1) if c else torch.zeros(n * self.H, dtype=torch.float64), 0.0)
            p = torch.where(see, (x - top[:, None]).exp(), 0.0)
            l = p.sum(1)
            w = p / l.clamp_min(1e-300)[:, None]
            vz = torch.nan_to_num(kv, nan=0.0)
            y, A = w @ vz, w @ vz.abs()
            dS = 576 * 2.0 ** -24 * abs(self.scale) * ((q.abs() @ kz.abs().T).amax(1) if c else torch.zeros(n * self.H, dtype=torch.float64))
            tol = 2.0 ** -8 * y.abs() + (2.0 ** -11 + 2 * dS)[:, None] * A + 2.0 ** -25 * (see.double() @ vz.abs()) / l.clamp_min(1.0)[:, None]
            got = out[at:at + n].cpu().double().reshape(n * self.H, 512) / out_scale
            ok = (got - y).abs() <= tol
            assert bool(ok[~poisoned & seen].all()), (b, float((got - y).abs()[~poisoned & seen].max()))
            assert not got[~seen].any()
            assert bool(torch.isnan(got[poisoned]).all())
            e = lse[at:at + n].cpu().double().reshape(-1)
            want = top + l.log()
            fine = seen & ~poisoned
            assert bool(((e - want).abs()[fine] <= (dS + 2.0 ** -20 + 2.0 ** -22 * want.abs())[fine]).all())
            assert bool((e[~seen] == -math.inf).all())
            at += n


CASES = [
    ([1], [1], 1, 64, True), ([1], [130], 64, 64, True), ([5], [5], 16, 64, False), ([3, 1, 7], [777, 64, 300], 16, 64, True),
    ([130], [130], 3, 16, True), ([64], [1000], 20, 128, True), ([2, 0, 33, 1], [2, 50, 520, 0], 5, 16, True),
    ([9], [700], 128, 64, True), ([1, 1, 1, 1, 1], [1, 255, 256, 257, 2000], 64, 64, True), ([40], [300], 7, 1, False),
    ([257], [513], 64, 64, True), ([100, 3], [100, 4097], 32, 256, True),
    # few rows per sequence, with every page size
    ([1], [300], 8, 1, True), ([2], [530], 4, 2, False), ([1, 1], [301, 65], 16, 4, True), ([3], [700], 16, 8, True),
    ([2], [900], 32, 32, False), ([1], [1300], 64, 4096, True), ([1, 4], [2050, 770], 16, 256, True),
    # more units than CTA pairs: several to a pair, cut anywhere
    ([150], [1500], 128, 64, True), ([1, 9, 2, 33, 1, 0, 17, 4] * 12, [300, 9, 700, 40, 1, 5, 260, 513] * 12, 32, 16, True),
    ([3] * 200, list(range(3, 203)), 64, 64, False),
]


@pytest.mark.parametrize("new,ctx,H,page,rope", CASES)
def test_prefill_matches_the_formula(new, ctx, H, page, rope):
    p = Problem(new, ctx, H, page, rope, seed=len(CASES) + sum(new))
    if sum(new) == 0:
        return
    # a sequence with more new tokens than context: its first tokens see nothing
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)


def test_rows_that_see_nothing():
    p = Problem([6, 4], [4, 0], 16, 16, True, seed=2)
    out, lse = p.run()
    p.check(out, lse)
    assert rt.device_errors() == 0


def test_missing_pages_are_masked_and_flagged():
    p = Problem([5, 3], [333, 100], 16, 16, True, seed=4)
    p.tables[0, 2], p.tables[0, 20], p.tables[1, :] = -1, p.pages, -1
    out, lse = p.run()
    assert rt.device_errors() == _lib.DEVERR_BAD_PAGE
    p.check(out, lse)


@pytest.mark.parametrize("gain,scale", [(8.0, 1.0 / 24.0), (1.0, -0.06), (1.0, 0.0), (64.0, 0.02)])
def test_scales_and_peaked_rows(gain, scale):
    p = Problem([33, 2], [900, 600], 16, 64, True, seed=6, q_gain=gain)
    p.scale = scale
    out, lse = p.run(bmm2_scale=0.5)
    p.check(out, lse, out_scale=0.5)


def test_rising_scores_move_the_maximum():
    """Later tokens score far above all earlier ones, tile after tile."""
    p = Problem([4], [1500], 16, 64, False, seed=8)
    g = torch.Generator().manual_seed(1)
    d = torch.randn(512, generator=g)
    x = torch.randn(p.pages * 64, 512, generator=g)
    slot = p.slots(0)
    x[slot] += d * torch.linspace(0, 4, 1500)[:, None]
    rt.write_nvfp4(x.to(torch.bfloat16).cuda(), p.pool, torch.arange(p.pages * 64, device="cuda"))
    p.q = (p.q.float() * 0.2 + torch.cat([d, torch.zeros(64)]).cuda()).to(torch.bfloat16)
    p.scale = 0.3
    out, lse = p.run()
    p.check(out, lse)


def test_hidden_bytes_do_not_reach_a_row():
    """Garbage (NaN scales, NaN rope rows) past the end of the sequences and in tokens that only
    later queries see."""
    p = Problem([70, 1], [200, 90], 16, 64, True, seed=10)
    raw, rope = p.pool.view(-1, 288), p.rope.view(-1, 64)
    live = torch.zeros(raw.shape[0], dtype=torch.bool)
    for b in range(2):
        live[p.slots(b)] = True
    raw[~live.cuda()] = 0xFF
    rope[~live.cuda()] = float("nan")
    p.pool[int(p.tables[0, 180 // 64]), 180 % 64, 256 + 5] = 0x7F       # token 180: one NaN block
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)


def test_strided_views_and_clamped_lengths():
    p = Problem([20, 13], [150, 77], 12, 16, True, seed=12)
    wide = torch.zeros(33, 12, 640, dtype=torch.bfloat16, device="cuda")
    wide[..., 64:] = p.q
    full = torch.zeros(33, 14, 520, dtype=torch.bfloat16, device="cuda")
    out, lse = p.run(q=wide[..., 64:], out=full[:, 1:13, 8:])
    p.check(out, lse)
    assert not full[:, 0].any() and not full[..., :8].any()
    # a sequence longer than max_seq_len is cut there and flagged
    cu = torch.tensor([0, 20, 33], dtype=torch.int32, device="cuda")
    seq = torch.tensor([150, 400], dtype=torch.int32, device="cuda")
    rt.mla_prefill(p.q, p.pool, None, 512, 64, p.tables.cuda(), cu, seq, 20, 150, bmm1_scale=p.scale)
    assert rt.device_errors() & _lib.DEVERR_SEQ_LEN


def test_far_pages():
    """Pool rows past 2^32 bytes."""
    p = Problem([3], [200], 16, 64, True, seed=14, spare=0)
    pages = (1 << 32) // (288 * 64) + 300
    pool = torch.zeros(pages, 64, 288, dtype=torch.uint8, device="cuda")
    rope = torch.zeros(pages, 64, 64, dtype=torch.bfloat16, device="cuda")
    far = pages - 1 - torch.arange(p.pages)
    pool[far.cuda()], rope[far.cuda()] = p.pool, p.rope
    out, lse = p.run()
    p.pool, p.rope, p.pages = pool, rope, pages
    p.tables = (pages - 1 - p.tables).int()
    got = p.run()
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_same_inputs_give_the_same_bits_and_other_streams():
    p = Problem([1, 40, 1], [3000, 500, 64], 32, 64, True, seed=16)
    out, lse = p.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = p.run()
    s.synchronize()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    p.check(out, lse)


def test_a_batch_whose_images_do_not_fit_runs_in_groups():
    """max_seq_len bounds the workspace: with a large one the batch takes several passes over it."""
    p = Problem([3, 40, 1], [300, 90, 1000], 16, 64, True, seed=18)
    out, lse = p.run()
    p.check(out, lse)
    most = 400000
    p.tables = torch.cat([p.tables, torch.full((3, most // 64 - p.width), -1, dtype=torch.int32)], 1)
    cu = torch.tensor([0, 3, 43, 44], dtype=torch.int32, device="cuda")
    seq = torch.tensor(p.ctx, dtype=torch.int32, device="cuda")
    again, lse2 = rt.mla_prefill(p.q, p.pool, None, 512, 64, p.tables.cuda(), cu, seq, 40, most, bmm1_scale=p.scale,
                                 rope_cache=p.rope, return_lse=True)
    assert rt.device_errors() == 0
    p.check(again, lse2)


@pytest.mark.parametrize("new,H", [(1, 64), (1, 33), (3, 20), (4, 20), (1, 1), (2, 65)])
def test_many_short_units(new, H):
    """Hundreds of units of one or two tiles, several to a CTA pair: 64 rows and fewer lie in both CTAs."""
    ctx = [new + (37 * i) % 460 for i in range(330)]
    p = Problem([new] * len(ctx), ctx, H, 16, True, seed=H)
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
    again = p.run(return_lse=False)
    assert torch.equal(out, again)


def test_device_errors_after_the_buffers_are_cleared():
    p = Problem([2], [70], 16, 16, False, seed=3)
    p.run()
    torch.cuda.synchronize()
    rt._bufs.clear()
    p.tables[0, 1] = -1
    out, lse = p.run()
    assert rt.device_errors() == _lib.DEVERR_BAD_PAGE
    p.check(out, lse)
