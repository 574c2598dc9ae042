"""GPU: the chunk attention with a sliding window and sinks against the formula in 64 bits.

The query at position p of its sequence sees tokens t <= p with t > p - W or t < S.  Tolerances as in
test_mla_prefill_gpu: the arithmetic of a row is the same over the tokens that it sees."""
import math

import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_gpu import Problem, latents

pytestmark = pytest.mark.gpu


class Windowed(Problem):
    def __init__(self, new, ctx, H, page, rope, window, sinks, trim=False, **kw):
        super().__init__(new, ctx, H, page, rope, **kw)
        self.W, self.S = window, sinks
        if trim:                # pages behind every window are gone
            for b, (n, c) in enumerate(zip(new, ctx)):
                for j in range(-(-c // page)):
                    if j * page >= sinks and (j + 1) * page <= c - n + 1 - window:
                        self.tables[b, j] = _lib.PAGE_TRIMMED if j % 2 else -1

    def run(self, **kw):
        return super().run(window=self.W, sinks=self.S, **kw)

    def check(self, out, lse, out_scale=1.0):
        at = 0
        for b, (n, c) in enumerate(zip(self.new, self.ctx)):
            R = n * self.H
            lo = max(0, c - n + 1 - self.W)
            t = torch.tensor([*range(min(self.S, lo, c)), *range(lo, c)], dtype=torch.long)     # what any row sees
            page = self.tables[b].long()[t // self.page]
            slot = torch.where((page >= 0) & (page < self.pages), page * self.page + t % self.page, -1)
            row, t, slot = slot.clamp_min(0).cuda(), t.cuda(), slot.cuda()
            kv = latents(self.pool.view(-1, 288)[row]).cuda()
            kr = self.rope.view(-1, 64)[row].double() if self.rope is not None else None
            q = self.q[at:at + n].double().reshape(R, 576)
            k = kv if kr is None else torch.cat([kv, kr], 1)
            q = q[:, : k.shape[1]]
            pos = (c - n + torch.arange(n, device="cuda")).repeat_interleave(self.H)[:, None]
            see = (t <= pos) & ((t > pos - self.W) | (t < self.S)) & (slot >= 0)
            kz = torch.nan_to_num(k, nan=0.0)
            x = torch.where(see, (q @ kz.T) * self.scale, -math.inf)
            poisoned = (see & torch.isnan(k).any(1)).any(1)
            seen = see.any(1)
            none = torch.zeros(R, dtype=torch.float64, device="cuda")
            top = torch.where(seen, x.amax(1) if t.numel() else none, 0.0)
            p = torch.where(see, (x - top[:, None]).exp(), 0.0)
            l = p.sum(1)
            w = p / l.clamp_min(1e-300)[:, None]
            vz = torch.nan_to_num(kv, nan=0.0)
            y, A = w @ vz, w @ vz.abs()
            dS = 576 * 2.0 ** -24 * abs(self.scale) * ((q.abs() @ kz.abs().T).amax(1) if t.numel() else none)
            tol = 2.0 ** -8 * y.abs() + (2.0 ** -11 + 2 * dS)[:, None] * A + 2.0 ** -25 * (see.double() @ vz.abs()) / l.clamp_min(1.0)[:, None]
            got = out[at:at + n].double().reshape(R, 512) / out_scale
            ok = (got - y).abs() <= tol
            assert bool(ok[~poisoned & seen].all()), (b, float((got - y).abs()[~poisoned & seen].max()))
            assert not got[~seen].any()
            assert bool(torch.isnan(got[poisoned]).all())
            e = lse[at:at + n].double().reshape(-1)
            want = top + l.log()
            fine = seen & ~poisoned
            assert bool(((e - want).abs()[fine] <= (dS + 2.0 ** -20 + 2.0 ** -22 * want.abs())[fine]).all())
            assert bool((e[~seen] == -math.inf).all())
            at += n


CASES = [
    # the smallest: a window of one token, one token, sinks past the sequence
    ([1], [1], 1, 64, True, 1, 0), ([1], [5], 64, 16, True, 1, 0), ([5], [5], 16, 64, False, 1, 1), ([3], [9], 4, 1, True, 2, 100),
    # windows and sinks at and around 64, 128 and 256
    ([1], [700], 64, 64, True, 64, 64), ([2], [1000], 64, 64, True, 65, 63), ([7], [777], 16, 64, False, 128, 4),
    ([1, 1, 1], [255, 256, 257], 64, 64, True, 128, 1), ([9], [1500], 128, 16, True, 255, 65), ([4], [1300], 32, 256, True, 256, 0),
    ([3, 1, 7], [777, 64, 300], 16, 64, True, 200, 129), ([40], [2000], 20, 64, True, 257, 200),
    # one head: a unit's rows are 128 tokens
    ([300], [1500], 1, 64, True, 100, 4), ([130], [130], 3, 16, True, 17, 5), ([257], [3000], 2, 128, False, 700, 300),
    # windows as long as the context, longer, and one token shorter
    ([10], [500], 16, 64, True, 500, 0), ([10], [500], 16, 64, True, 1 << 40, 1 << 40), ([10], [500], 16, 64, True, 499, 0),
    # rows that see nothing (more new tokens than context), empty sequences
    ([6, 4], [4, 0], 16, 16, True, 2, 1), ([2, 0, 33, 1], [2, 50, 520, 0], 5, 16, True, 40, 7),
    # chunks that begin before their window is full
    ([600], [600], 16, 64, True, 128, 4), ([900, 1], [950, 4000], 8, 64, True, 300, 70),
    # units cut between CTA pairs, more units than pairs
    ([150], [5000], 128, 64, True, 1100, 64), ([1], [9000], 64, 64, True, 4096, 4),
    ([1, 9, 2, 33, 1, 0, 17, 4] * 12, [300, 9, 700, 40, 1, 5, 260, 513] * 12, 32, 16, True, 90, 3),
    ([3] * 200, list(range(3, 203)), 64, 64, False, 31, 2),
]


# calls of more than two 128-token tiles of 64 rows an SM: the chunk kernel's own form
LARGE = [
    ([400], [1500], 64, 64, True, 1, 0), ([300], [700], 64, 16, True, 64, 64), ([129], [1000], 128, 64, True, 65, 63),
    ([700], [777], 20, 64, False, 128, 4), ([100, 100, 100], [255, 256, 257], 64, 64, True, 128, 1), ([260], [1500], 128, 16, True, 255, 65),
    ([300], [1300], 64, 256, True, 256, 0), ([300, 1, 70], [777, 64, 300], 64, 64, True, 200, 129), ([1100], [3000], 20, 64, True, 257, 200),
    ([2900], [3000], 1, 64, True, 700, 300), ([640], [640], 64, 16, True, 17, 5), ([500], [500], 64, 64, True, 499, 0),
    ([600, 300], [400, 0], 64, 16, True, 200, 100), ([70, 0, 233, 1], [70, 50, 520, 0], 65, 16, True, 40, 7), ([200], [9000], 64, 64, True, 4096, 4),
    ([129, 3, 1, 77] * 3, [5000, 3, 900, 300] * 3, 32, 1, True, 1000, 128),
]


@pytest.mark.parametrize("new,ctx,H,page,rope,window,sinks", LARGE)
def test_large_calls_match_the_formula(new, ctx, H, page, rope, window, sinks):
    span = min(max(new), (H + 62) // H + 1)
    tiles = -(-min(sinks + window - 1 + span, max(ctx)) // 128)
    assert len(new) * -(-max(new) * H // 64) * tiles > 2 * torch.cuda.get_device_properties(0).multi_processor_count
    p = Windowed(new, ctx, H, page, rope, window, sinks, trim=True, seed=sum(new))
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
    again = p.run()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("new,ctx,H,page,rope,window,sinks", CASES)
def test_window_matches_the_formula(new, ctx, H, page, rope, window, sinks, trim):
    p = Windowed(new, ctx, H, page, rope, window, sinks, trim=trim, seed=len(CASES) + sum(new))
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)


def test_a_window_that_hides_nothing_gives_the_same_bits():
    p = Windowed([40, 1], [700, 300], 16, 64, True, 699, 1, seed=3)
    a = p.run()
    b = Problem.run(p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_the_longest_windows_and_sinks():
    """Positions before a sequence's start (length 5 with 60 new tokens) less a window of nearly 2^31."""
    most = 2 ** 31 - 1
    for window, sinks in ((most - 50, 0), (most - 50, 20), (1, most - 50), (700, most - 800)):
        p = Windowed([60, 3], [5, 900], 1, 1024, True, window, sinks, seed=6)
        tables = torch.full((2, 1 << 21), -1, dtype=torch.int32, device="cuda")
        tables[:, : p.tables.shape[1]] = p.tables
        cu = torch.tensor([0, 60, 63], dtype=torch.int32, device="cuda")
        out, lse = rt.mla_prefill(p.q, p.pool, None, 512, 64, tables, cu, torch.tensor(p.ctx, dtype=torch.int32, device="cuda"),
                                  60, most, bmm1_scale=p.scale, rope_cache=p.rope, return_lse=True, window=window, sinks=sinks)
        assert rt.device_errors() == 0
        p.check(out, lse)


@pytest.mark.parametrize("n,H", [(5, 16), (90, 128)])
def test_missing_pages_in_and_behind_the_window(n, H):
    p = Windowed([n, 3], [900, 600], H, 16, True, 100, 20, seed=4)
    # sequence 0: sinks on pages 0 and 1, windows from token 801 - n on
    p.tables[0, 2:(801 - n) // 16] = -1
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
    for j in (1, 52):
        keep = p.tables.clone()
        p.tables[0, j] = p.pages if j == 1 else _lib.PAGE_TRIMMED
        out, lse = p.run()
        assert rt.device_errors() == _lib.DEVERR_BAD_PAGE
        p.check(out, lse)
        p.tables = keep


@pytest.mark.parametrize("H", [16, 128])
def test_hidden_bytes_do_not_reach_a_row(H):
    """NaN latents and rope rows in every token that no row sees, and one that only some rows see."""
    p = Windowed([70, 1], [900, 2000], H, 64, True, 150, 5, seed=10)
    raw, rope = p.pool.view(-1, 288), p.rope.view(-1, 64)
    live = torch.zeros(raw.shape[0], dtype=torch.bool)
    for b, (n, c) in enumerate(zip(p.new, p.ctx)):
        live[p.slots(b)[[*range(5), *range(c - n + 1 - 150, c)]]] = True
    raw[~live.cuda()] = 0xFF
    rope[~live.cuda()] = float("nan")
    p.pool[int(p.tables[0, 700 // 64]), 700 % 64, 256 + 5] = 0x7F       # token 700: seen by the first rows only
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)


@pytest.mark.parametrize("n,H", [(33, 16), (150, 64)])
@pytest.mark.parametrize("gain,scale", [(8.0, 1.0 / 24.0), (1.0, -0.06), (1.0, 0.0), (64.0, 0.02)])
def test_scales_and_peaked_rows(gain, scale, n, H):
    p = Windowed([n, 2], [900, 600], H, 64, True, 300, 10, seed=6, q_gain=gain)
    p.scale = scale
    out, lse = p.run(bmm2_scale=0.5)
    p.check(out, lse, out_scale=0.5)


def test_a_batch_whose_images_do_not_fit_runs_in_groups():
    """The images' bound is 1 GiB: 400 sequences' windows of 1,000 tokens, 3 MB each, take two passes."""
    n = 400
    p = Windowed([2] * n, [1100 + (7 * i) % 400 for i in range(n)], 64, 64, False, 1000, 4, seed=18)
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)


@pytest.mark.parametrize("H", [12, 600])
def test_clamped_lengths_and_padding_rows(H):
    """Sequences past the bounds end there, flagged; rows of no sequence stay as they were."""
    p = Windowed([20, 13], [400, 377], H, 16, True, 60, 4, seed=12)
    out, lse = p.run()
    p.check(out, lse)
    cu = torch.tensor([0, 20, 33], dtype=torch.int32, device="cuda")
    seq = torch.tensor([400, 377], dtype=torch.int32, device="cuda")
    q = torch.cat([p.q, p.q[:5]])
    full = torch.full((38, H, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    rt.mla_prefill(q, p.pool, None, 512, 64, p.tables.cuda(), cu, seq, 20, 400, out=full, bmm1_scale=p.scale, rope_cache=p.rope,
                   window=60, sinks=4)
    assert rt.device_errors() == 0
    assert torch.equal(full[:33], out) and bool((full[33:] == 7.0).all())
    # only the first 13 new tokens are computed: each as in the whole chunk
    full.fill_(7.0)
    rt.mla_prefill(q, p.pool, None, 512, 64, p.tables.cuda(), cu, seq, 13, 400, out=full, bmm1_scale=p.scale, rope_cache=p.rope,
                   window=60, sinks=4)
    assert rt.device_errors() == _lib.DEVERR_SEQ_LEN
    assert bool((full[13:20] == 7.0).all()) and bool((full[33:] == 7.0).all())
    p.check(torch.cat([full[:13], out[13:20], full[20:33]]), lse)
    # none of them, and none at all
    full.fill_(7.0)
    rt.mla_prefill(q, p.pool, None, 512, 64, p.tables.cuda(), cu, seq, 0, 400, out=full, bmm1_scale=p.scale, window=60)
    assert rt.device_errors() == _lib.DEVERR_SEQ_LEN and bool((full == 7.0).all())
    rt.mla_prefill(q, p.pool, None, 512, 64, p.tables.cuda(), cu * 0, seq, 20, 400, out=full, bmm1_scale=p.scale, window=60)
    assert rt.device_errors() == 0 and bool((full == 7.0).all())


def test_chunks_and_one_pass_agree():
    """A token's row is the same sum over the same tokens in both, with other references for its
    probabilities, whose 11 bits are then cut elsewhere: each pass is within 2^-8 |y| + (2^-11 + 2 dS) A
    of the formula (test_mla_prefill_gpu; A at most the largest |v|), so the two within twice that."""
    p = Windowed([1000], [1000], 16, 64, False, 200, 4, seed=3)
    out, lse = p.run()
    parts = []
    for lo in range(0, 1000, 130):
        hi = min(lo + 130, 1000)
        parts.append(rt.mla_prefill(p.q[lo:hi], p.pool, None, 512, 64, p.tables.cuda(),
                                    torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"),
                                    torch.tensor([hi], dtype=torch.int32, device="cuda"), hi - lo, hi, bmm1_scale=p.scale,
                                    return_lse=True, window=200, sinks=4))
    again, lse2 = (torch.cat(v) for v in zip(*parts))
    p.check(out, lse)
    p.check(again, lse2)
    v = latents(p.pool.view(-1, 288)).abs()
    dS = 576 * 2.0 ** -24 * p.scale * float((p.q[..., :512].abs().double().cpu().reshape(-1, 512) @ v.T).max())
    whole = out.double()
    assert bool(((whole - again.double()).abs() <= 2.0 ** -7 * whole.abs() + (2.0 ** -10 + 4 * dS) * float(v.max())).all())
    assert rt.device_errors() == 0


@pytest.mark.parametrize("H", [32, 128])
def test_a_graph_follows_the_lengths_on_the_device(H):
    p = Windowed([4, 6], [900, 1200], H, 64, True, 300 if H == 32 else 1100, 10, seed=5)
    cu = torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda")
    seq = torch.tensor([900, 1200], dtype=torch.int32, device="cuda")
    tables = p.tables.cuda()
    out = torch.empty(10, H, 512, dtype=torch.bfloat16, device="cuda")
    call = lambda: rt.mla_prefill(p.q, p.pool, None, 512, 64, tables, cu, seq, 8, 1216, out=out, bmm1_scale=p.scale,  # noqa: E731
                                  rope_cache=p.rope, window=p.W, sinks=10)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
    for lens, starts in (([900, 1200], [0, 4, 10]), ([33, 1200], [0, 1, 9]), ([900, 5], [0, 8, 10])):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got[: starts[-1]], out[: starts[-1]])
        assert bool((got[starts[-1]:] == 7.0).all())
    assert rt.device_errors() == 0


# units of up to 64 rows in 2 to 8 parts each, with enough of them to fill most of the SMs; shorter sequences
# among them have fewer parts, one or none
JOINED = [
    ([1] * 64, [250, 64, 1, 700] * 16, 64, 64, True, 200, 4), ([3] * 30, [900, 500, 3, 2, 0, 260] * 5, 20, 16, True, 500, 0),
    ([1] * 15, [1100, 1500, 600] * 5, 64, 64, True, 1000, 20), ([1] * 24, [700, 130, 4000, 512] * 6, 64, 256, True, 600, 10),
    ([64] * 37, [600] * 30 + [64, 100, 200, 300, 30, 0, 1], 1, 64, False, 300, 1), ([1, 0] * 50, [300, 300, 200, 64] * 25, 8, 1, True, 250, 4),
    ([8] * 4, [500, 2000, 505, 700], 64, 64, True, 500, 0), ([1] * 19, [1300, 900] * 9 + [40], 63, 64, True, 800, 70),
]


@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("new,ctx,H,page,rope,window,sinks", JOINED)
def test_many_units_of_several_parts(new, ctx, H, page, rope, window, sinks, trim):
    p = Windowed(new, ctx, H, page, rope, window, sinks, trim=trim, seed=len(new))
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
    for _ in range(5):
        again = p.run()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_missing_pages_and_nan_scales_in_some_parts():
    p = Windowed([1] * 64, [250, 200, 255, 256] * 16, 64, 16, True, 250, 4, seed=8)
    p.pool.view(-1, 288)[p.slots(3)[17], 256] = 0x7F        # a token of sequence 3's first part
    p.tables[5, 12] = -1                                    # tokens 192 .. 207: the second part of sequence 5
    p.tables[9, :8] = p.pages                               # all but what lies behind the window of its first part
    out, lse = p.run()
    assert rt.device_errors() == _lib.DEVERR_BAD_PAGE
    p.check(out, lse)


def test_what_follows_a_call_without_parts_reads_its_output():
    """Tables wide enough for several parts of a unit, sequences short enough for one: nothing is merged,
    and the next kernels still find the output."""
    p = Windowed([1] * 8, [100, 1, 128, 77, 5, 120, 64, 90], 64, 64, True, 1000, 4, seed=21)
    cu = torch.arange(9, dtype=torch.int32, device="cuda")
    seq = torch.tensor(p.ctx, dtype=torch.int32, device="cuda")
    tables = torch.nn.functional.pad(p.tables.cuda(), (0, 64), value=-1)
    first = None
    for _ in range(200):
        out = torch.full((8, 64, 512), 7.0, dtype=torch.bfloat16, device="cuda")
        rt.mla_prefill(p.q, p.pool, None, 512, 64, tables, cu, seq, 1, 4096, out=out, bmm1_scale=p.scale, rope_cache=p.rope, window=1000, sinks=4)
        after = out.clone()
        first = after if first is None else first
        assert torch.equal(after, first)
    p.check(first, p.run()[1])


def test_long_context():
    """A window at the end of 300,000 tokens whose other pages are gone."""
    p = Windowed([3], [1000], 16, 64, True, 600, 20, seed=21)
    out, lse = p.run()
    p.check(out, lse)
    # the same sequence with 4,672 pages put between its first page and its sixth
    far = torch.full((1, 16 + 4672), _lib.PAGE_TRIMMED, dtype=torch.int32)
    far[0, 0] = p.tables[0, 0]
    far[0, 6 + 4672: 16 + 4672] = p.tables[0, 6:16]
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    seq = torch.tensor([1000 + 4672 * 64], dtype=torch.int32, device="cuda")
    got = rt.mla_prefill(p.q, p.pool, None, 512, 64, far.cuda(), cu, seq, 3, 300032, bmm1_scale=p.scale, rope_cache=p.rope,
                         return_lse=True, window=600, sinks=20)
    assert rt.device_errors() == 0
    p.check(got[0], got[1])


@pytest.mark.parametrize("change,word", [(dict(window=-1), "window"), (dict(window=4, sinks=-1), "window"), (dict(sinks=3), "window")])
def test_refusals(change, word):
    p = Problem([1], [20], 4, 16, True)
    with pytest.raises(ValueError, match=word):
        p.run(**change)
