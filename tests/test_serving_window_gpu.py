"""GPU: a step's tables, rotary positions with several axes, attention with a window, and giving back
the pages behind it, together: as the serving loop calls them, as one captured graph, and against the
same sequences kept whole."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from glm53_flash_dual_dgx_spark_b200 import serving_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,prompt,window,sinks,image", [(64, 700, 0, 0, True), (64, 700, 200, 4, False), (16, 900, 64, 70, True), (5, 64, 500, 0, True)])
def test_serving_loop(heads, prompt, window, sinks, image):
    got = serving_step.run(heads=heads, prompt=prompt, steps=2, window=window, sinks=sinks, image=image)
    assert got["device_errors"] == 0
    assert got["fork_equals_parent"] and got["compaction_keeps_outputs"]
    assert got["highest_page"] == got["live_pages"] - 1
    assert not torch.isnan(got["out"]).any()
    whole = serving_step.run(heads=heads, prompt=prompt, steps=2, image=image)
    if window and prompt > window + 2 * 64:
        assert got["live_pages"] < whole["live_pages"] and got["shared_pages"] < whole["shared_pages"]
    assert torch.equal(got["out"], whole["out"]) == (not window or prompt <= window)


@pytest.mark.parametrize("window", [255, 256])
def test_serving_loop_wherever_the_window_begins_in_a_page(window):
    for prompt in range(500, 564, 3):
        got = serving_step.run(heads=2, prompt=prompt, steps=3, window=window, sinks=4)
        assert got["device_errors"] == 0 and got["fork_equals_parent"] and got["compaction_keeps_outputs"], prompt
    got = serving_step.run(heads=2, prompt=700, steps=3, window=256, sinks=4)
    assert got["device_errors"] == 0


class Twin:
    """The same growing sequences twice: with pages placed on the device and trimmed behind the window, and
    in a pool where every sequence has its pages for good."""

    def __init__(self, lens, most, page, H, window, sinks, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.page, self.H, self.seen, B = page, H, dict(window=window, sinks=sinks), len(lens)
        width = -(-most // page)
        pool = lambda n: (torch.zeros(n, page, 288, dtype=torch.uint8, device="cuda"), torch.zeros(n, page, 64, dtype=torch.bfloat16, device="cuda"))  # noqa: E731
        self.cache, self.whole = pool(B * width // 2 + 2 * B), pool(B * width)
        self.refs = torch.zeros(self.cache[0].shape[0], dtype=torch.int32, device="cuda")
        self.tables = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
        self.all = torch.randperm(B * width, generator=self.g, device="cuda").view(B, width).int()
        self.lens, self.host = torch.zeros(B, dtype=torch.int32, device="cuda"), [0] * B
        self.cos_sin, self.axes = rt.rope_cos_sin(4096).cuda(), rt.rope_axes((8, 12, 12))

    def step(self, slots, new, keep):
        """The sequences in `slots`, cut back to `keep` tokens, grow by `new`."""
        T, dev = sum(new), "cuda"
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        draw = lambda *s: torch.randn(*s, generator=self.g, device=dev).to(torch.bfloat16)  # noqa: E731
        q, kv, kr = draw(T, self.H, 576), draw(T, 512), draw(T, 64)
        e = rt.extend_pages(self.tables, self.lens, ints(slots), ints(new), self.refs, self.page, T + 3, lens=ints(keep))
        pos = torch.cat([torch.arange(k, k + n, device=dev) for k, n in zip(keep, new)])
        assert torch.equal(e.positions[:T].long(), pos) and bool((e.slot_mapping[T:] == -1).all())
        axes = torch.stack([pos, pos // 7, pos % 13])
        seq = torch.tensor(slots, device=dev).repeat_interleave(torch.tensor(new, device=dev))
        home = self.all[seq, pos // self.page].long() * self.page + pos % self.page
        cu = ints([sum(new[:k]) for k in range(len(new) + 1)])
        outs = []
        for (latent, rope), slot, tables, starts, lens, rows in (
                (self.cache, e.slot_mapping, e.block_tables, e.cu_seqlens_q, e.seq_lens, T + 3),
                (self.whole, home, self.all[torch.tensor(slots, device=dev)], cu, ints([k + n for k, n in zip(keep, new)]), T)):
            pad = lambda x: torch.cat([x, x.new_zeros(rows - T, *x.shape[1:])])  # noqa: E731
            q2 = pad(q)
            rt.write_nvfp4(pad(kv), latent, slot)
            rt.write_nvfp4_rope_rotated(pad(kr), rope, slot, torch.cat([axes, axes.new_zeros(3, rows - T)], 1), self.cos_sin,
                                        q_pe=q2[..., 512:], axes=self.axes)
            outs.append(rt.mla_prefill(q2, latent, None, 512, 64, tables, starts, lens, max(new), self.tables.shape[1] * self.page,
                                       bmm1_scale=1 / 24, rope_cache=rope, return_lse=True, **self.seen))
        assert torch.equal(outs[0][0][:T], outs[1][0]) and torch.equal(outs[0][1][:T], outs[1][1])
        rt.trim_pages(self.tables, self.lens, ints(slots), self.refs, self.page, window=self.seen["window"] + 5, sinks=self.seen["sinks"])
        assert rt.device_errors() == 0


@pytest.mark.parametrize("page,H,window,sinks", [(16, 8, 50, 5), (64, 64, 130, 0), (16, 20, 1, 40)])
def test_trimmed_sequences_give_what_whole_ones_give(page, H, window, sinks):
    """Chunks, drafts of which some are taken back, and single tokens: the same bits from a pool half as
    large, in which pages are given back and placed again."""
    t = Twin([0, 0, 0], 600, page, H, window, sinks, seed=page + H)
    t.step([0, 1, 2], [200, 17, 90], [0, 0, 0])
    t.step([2, 0], [100, 150], [90, 200])
    t.step([1, 0, 2], [60, 5, 5], [17, 350, 190])
    t.step([0, 2, 1], [5, 5, 5], [352, 195, 73])       # 3, 0 and 4 of the last tokens taken back
    for i in range(6):
        t.step([0, 1, 2], [1, 1, 1], [357 + i, 78 + i, 200 + i])
    t.step([1], [300], [80])
    live = int((t.refs > 0).sum())
    assert live <= sum(-(-(min(n, window + 5) + sinks) // page) + 2 for n in (363, 380, 206))


@pytest.mark.parametrize("H,window", [(64, 900), (64, 100), (128, 900)])
def test_attention_right_behind_the_tables(H, window):
    """Steps whose lengths change by hundreds of tokens, nothing between their tables and the attention, and
    nothing waited for: each as with a wait."""
    g = torch.Generator(device="cuda").manual_seed(H + window)
    B, page, pages = 4, 64, 80
    latent = torch.zeros(pages, page, 288, dtype=torch.uint8, device="cuda")
    rt.write_nvfp4(torch.randn(pages * page, 512, generator=g, device="cuda").to(torch.bfloat16), latent, torch.arange(pages * page, device="cuda"))
    q = torch.randn(2 * B, H, 576, generator=g, device="cuda").to(torch.bfloat16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    slots = ints([0, 1, 2, 3])
    rows = [(ints([1 + (i + k) % 2 for k in range(B)]), ints([(37 * i + 311 * k) % 1100 for k in range(B)])) for i in range(24)]

    def run(wait):
        tables, lens, refs = torch.full((B, 18), -1, dtype=torch.int32, device="cuda"), ints([0] * B), ints([0] * pages)
        rt.extend_pages(tables, lens, slots, ints([1140] * B), refs, page, 4 * 1140)
        start, outs = [t.clone() for t in (tables, lens, refs)], []
        torch.cuda.synchronize()
        for new, keep in rows:
            for t, t0 in zip((tables, lens, refs), start):
                t.copy_(t0)
            e = rt.extend_pages(tables, lens, slots, new, refs, page, 2 * B, lens=keep)
            if wait:
                torch.cuda.synchronize()
            outs.append(rt.mla_prefill(q, latent, None, 512, 64, e.block_tables, e.cu_seqlens_q, e.seq_lens, 2, 1152,
                                       bmm1_scale=1 / 24, return_lse=True, window=window, sinks=3))
            if wait:
                torch.cuda.synchronize()
        return outs

    want, got = run(True), run(False)
    assert rt.device_errors() == 0
    for i, ((a, al), (b, bl)) in enumerate(zip(want, got)):
        n = int(rows[i][0].sum())
        assert torch.equal(a[:n], b[:n]) and torch.equal(al[:n], bl[:n])


def test_a_step_in_one_graph():
    """extend, rotate and write, attend, trim, captured once and replayed as the sequences grow."""
    page, H, window, sinks, T = 16, 16, 40, 5, 12
    g = torch.Generator(device="cuda").manual_seed(4)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    latent, rope = torch.zeros(30, page, 288, dtype=torch.uint8, device="cuda"), torch.zeros(30, page, 64, dtype=torch.bfloat16, device="cuda")
    tables, lens, refs = torch.full((3, 20), -1, dtype=torch.int32, device="cuda"), ints(0, 0, 0), torch.zeros(30, dtype=torch.int32, device="cuda")
    slots, new, keep = ints(0, 1, 2), ints(4, 4, 4), ints(0, 0, 0)
    cos_sin, axes = rt.rope_cos_sin(512).cuda(), rt.rope_axes((16, 16))
    q0, kv, kr, q = draw(T, H, 576), draw(T, 512), draw(T, 64), torch.empty(T, H, 576, dtype=torch.bfloat16, device="cuda")
    state = [latent, rope, tables, lens, refs]

    def step():
        q.copy_(q0)
        e = rt.extend_pages(tables, lens, slots, new, refs, page, T, lens=keep)
        rt.write_nvfp4(kv, latent, e.slot_mapping)
        rt.write_nvfp4_rope_rotated(kr, rope, e.slot_mapping, torch.stack([e.positions, e.positions // 3]), cos_sin, q_pe=q[..., 512:], axes=axes)
        out = rt.mla_prefill(q, latent, None, 512, 64, e.block_tables, e.cu_seqlens_q, e.seq_lens, T, 320, bmm1_scale=1 / 24,
                             rope_cache=rope, window=window, sinks=sinks)
        rt.trim_pages(tables, lens, slots, refs, page, window=window + 2, sinks=sinks)      # (up to 2 tokens are taken back)
        return out

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        s.synchronize()
        start = [t.clone() for t in state]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
        rows = [((4, 4, 4), (4, 2, 0)), ((10, 1, 1), (8, 6, 4)), ((1, 9, 2), (18, 5, 3)), ((12, 0, 0), (19, 14, 5)), ((1, 1, 1), (31, 14, 5))] \
            + [((1, 1, 1), (32 + i, 15 + i, 6 + i)) for i in range(60)]
        want = []
        for n, k in rows:
            new.copy_(ints(*n)), keep.copy_(ints(*k))
            want.append(step()[: sum(n)].clone())
        assert rt.device_errors() == 0 and tables[0, 1:4].tolist()[:2] == [-2, -2]      # 92 tokens: pages 1 and 2 end before 92 - 41
        for t, t0 in zip(state, start):
            t.copy_(t0)
        for (n, k), w in zip(rows, want):
            new.copy_(ints(*n)), keep.copy_(ints(*k))
            graph.replay()
            s.synchronize()
            assert torch.equal(out[: sum(n)], w)
    assert rt.device_errors() == 0
