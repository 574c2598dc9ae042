"""GPU: windowed chunk attention in each of its forms, told apart by the kernels of a captured call: few
rows in one part a unit (one kernel), in parts merged by a second kernel (two), in parts that merge in
their cluster (one), and large calls (an image, the attention, the merge of cut units: three)."""
import pytest
import torch
from cuda.bindings import runtime as cudart

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_window_gpu import Windowed

pytestmark = pytest.mark.gpu


def kernels(call) -> int:
    """Kernels of a call, once it has run."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph, stream=s):
            call()
    err, _, num = cudart.cudaGraphGetNodes(graph.raw_cuda_graph())
    assert err == cudart.cudaError_t.cudaSuccess
    err, nodes, num = cudart.cudaGraphGetNodes(graph.raw_cuda_graph(), num)
    types = [cudart.cudaGraphNodeGetType(n)[1] for n in nodes[:num]]
    return types.count(cudart.cudaGraphNodeType.cudaGraphNodeTypeKernel)


def device_call(p):
    """p.run with its lengths and tables on the device beforehand."""
    cu = torch.tensor([sum(p.new[:b]) for b in range(len(p.new) + 1)], dtype=torch.int32, device="cuda")
    seq, tables = torch.tensor(p.ctx, dtype=torch.int32, device="cuda"), p.tables.cuda()
    return lambda: rt.mla_prefill(p.q, p.pool, None, 512, 64, tables, cu, seq, max(p.new), max(p.ctx), bmm1_scale=p.scale,
                                  rope_cache=p.rope, return_lse=True, window=p.W, sinks=p.S)


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def plan(p):
    """Units of 64 rows and parts a unit, of a call whose rows are few; parts 0 for a large one."""
    longest, few_units = max(p.new), -(-max(p.new) * p.H // 64)
    span, units = min(longest, (p.H + 62) // p.H + 1), few_units * len(p.new)
    tiles = -(-min(p.S + p.W - 1 + span, max(p.ctx)) // 128)
    if few_units > 1 and units > 2 * sms() // tiles:
        return units, 0
    return units, min(max(sms() // units, 1), 64, tiles)


# single tokens in clusters of eight parts, and among them sequences of six or seven: a CTA there merges up to ten or
# twelve pieces, eight at a time
@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("new,ctx,H,rope", [
    ([1] * 15, [1100, 700, 800, 896, 2000] * 3, 64, True), ([1] * 15, [641, 768, 769, 897, 1005] * 3, 64, False),
    ([3] * 15, [900, 3, 702, 1500, 770] * 3, 20, True), ([1] * 14, [700] * 13 + [5000], 63, True)])
def test_units_of_fewer_parts_than_their_cluster(new, ctx, H, rope, trim):
    p = Windowed(new, ctx, H, 64, rope, 1000, 4, trim=trim, seed=sum(ctx))
    units, parts = plan(p)
    assert parts == 8 and 8 * units * parts >= 5 * sms()
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
    assert kernels(device_call(p)) == 1
    for _ in range(5):
        again = p.run()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_missing_pages_and_nan_scales_in_units_of_fewer_parts():
    p = Windowed([1] * 15, [1100, 700, 800, 896, 650] * 3, 64, 16, True, 1000, 4, seed=3)
    p.pool.view(-1, 288)[p.slots(1)[600], 256] = 0x7F       # a token of sequence 1's last part
    p.pool.view(-1, 288)[p.slots(3)[17], 256 + 31] = 0x7F   # a token of sequence 3's first part
    p.tables[6, 8:40] = -1                                  # tokens 128 .. 639 of 700: parts 1 to 4 of sequence 6
    p.tables[7, 49] = p.pages
    out, lse = p.run()
    assert rt.device_errors() == _lib.DEVERR_BAD_PAGE
    p.check(out, lse)
    assert kernels(device_call(p)) == 1
    rt.device_errors()


FORMS = [      # (the case, its kernels)
    ([7, 1], [90, 70], 9, 50, 3, 1), ([1, 4], [700, 500], 64, 300, 4, 2), ([2, 3], [900, 500], 16, 700, 5, 2),
    ([1] * 50, [300, 250, 100, 500, 260] * 10, 64, 250, 4, 1), ([150, 40], [900, 41], 64, 300, 70, 3), ([300], [1500], 64, 400, 0, 3),
]


@pytest.mark.parametrize("new,ctx,H,window,sinks,num", FORMS)
def test_the_forms_match_the_formula(new, ctx, H, window, sinks, num):
    p = Windowed(new, ctx, H, 64, True, window, sinks, trim=True, seed=num)
    assert (plan(p)[1] == 0) == (num == 3)
    out, lse = p.run()
    assert kernels(device_call(p)) == num
    p.check(out, lse)


@pytest.mark.parametrize("new,ctx,H,window,sinks,num", FORMS)
def test_strided_views(new, ctx, H, window, sinks, num):
    """Queries between other heads and dims, or head by head; outputs there, on 16- and on 32-byte
    boundaries; tables that are a view: the bits of the contiguous call, and nothing written beside them."""
    p = Windowed(new, ctx, H, 64, True, window, sinks, seed=num)
    want, lse = p.run()
    T = sum(new)
    big = torch.full((T, H + 3, 640), float("nan"), dtype=torch.bfloat16, device="cuda")
    queries = [big[:, 2:H + 2, 8:584], torch.empty(H, T, 576, dtype=torch.bfloat16, device="cuda").transpose(0, 1)]
    tables = torch.full((2 * len(new), p.width + 9), p.pages, dtype=torch.int32, device="cuda")[::2, 5:5 + p.width]
    tables.copy_(p.tables)
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    seq = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    for q in queries:
        q.copy_(p.q)
        for first, step in ((8, 528), (16, 528), (8, 520), (0, 512)):
            for by_head in (False, True):
                shape = (H + 2, T, step) if by_head else (T, H + 2, step)
                room = torch.full((shape[0] * shape[1] * step + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
                whole = room[first:first + shape[0] * shape[1] * step].view(shape)
                out = (whole.transpose(0, 1) if by_head else whole)[:, 1:H + 1, :512]
                got = rt.mla_prefill(q, p.pool, None, 512, 64, tables, cu, seq, max(new), max(ctx), out=out, bmm1_scale=p.scale,
                                     rope_cache=p.rope, return_lse=True, window=window, sinks=sinks)
                assert got[0].data_ptr() == out.data_ptr()
                assert torch.equal(out, want) and torch.equal(got[1], lse)
                out.fill_(7.0)
                assert bool((room == 7.0).all())
    assert rt.device_errors() == 0


@pytest.mark.parametrize("new,ctx,H,window,sinks,num", FORMS)
def test_queries_that_are_not_finite(new, ctx, H, window, sinks, num):
    """A NaN or an infinity makes its own row NaN (some visible score is NaN or +inf), and no other."""
    p = Windowed(new, ctx, H, 64, True, window, sinks, seed=num)
    want, lse = p.run()
    inf, nan = float("inf"), float("nan")
    bad = []
    for k, (dim, value) in enumerate(((0, nan), (511, inf), (200, -inf), (512, nan), (575, inf), (530, -inf), (64, nan))):
        row = (k * 131) % (sum(new) * H)
        if row not in bad:
            bad.append(row)
            p.q[row // H, row % H, dim] = value
    out, e = p.run()
    flat, ok = out.view(-1, 512), torch.ones(sum(new) * H, dtype=torch.bool, device="cuda")
    ok[bad] = False
    assert len(bad) >= 5
    # (every one of these rows sees enough tokens that an infinite query meets a zero or a value of its sign)
    assert bool(torch.isnan(flat[~ok]).all()) and not bool(torch.isfinite(e.view(-1)[~ok]).any())
    assert torch.equal(flat[ok], want.view(-1, 512)[ok]) and torch.equal(e.view(-1)[ok], lse.view(-1)[ok])
    assert rt.device_errors() == 0


def test_a_graph_of_large_calls_follows_the_lengths_on_the_device():
    p = Windowed([150, 160], [900, 1200], 64, 64, True, 300, 10, seed=5)
    assert plan(p)[1] == 0
    cu = torch.tensor([0, 150, 310], dtype=torch.int32, device="cuda")
    seq = torch.tensor([900, 1200], dtype=torch.int32, device="cuda")
    tables = p.tables.cuda()
    out, lse = torch.empty(310, 64, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(310, 64, device="cuda")

    def call():
        lse.copy_(rt.mla_prefill(p.q, p.pool, None, 512, 64, tables, cu, seq, 160, 1216, out=out, bmm1_scale=p.scale,
                                 rope_cache=p.rope, return_lse=True, window=300, sinks=10)[1])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
    for lens, starts in (([900, 1200], [0, 150, 310]), ([33, 1200], [0, 33, 190]), ([900, 5], [0, 160, 165]), ([0, 700], [0, 0, 90]),
                         ([500, 0], [0, 1, 1]), ([900, 1200], [0, 150, 310])):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, e = out.clone(), lse.clone()
        call()
        torch.cuda.synchronize()
        n = starts[-1]
        assert torch.equal(got[:n], out[:n]) and torch.equal(e[:n], lse[:n])
        assert bool((got[n:] == 7.0).all())
        # (and it is what these lengths give)
        q = p.q
        p.q, p.new, p.ctx = q[:n], [starts[1], starts[2] - starts[1]], lens
        p.check(got[:n], e[:n])
        p.q = q
    assert rt.device_errors() == 0


@pytest.mark.parametrize("H,window", [(64, 300), (128, 900)])
def test_large_calls_right_behind_the_tables(H, window):
    """Steps of chunks whose lengths change by hundreds of tokens, nothing between their tables and the
    attention, and nothing waited for: each as with a wait."""
    g = torch.Generator(device="cuda").manual_seed(H + window)
    B, page, pages, T = 4, 64, 90, 360
    latent = torch.zeros(pages, page, 288, dtype=torch.uint8, device="cuda")
    rt.write_nvfp4(torch.randn(pages * page, 512, generator=g, device="cuda").to(torch.bfloat16), latent, torch.arange(pages * page, device="cuda"))
    q = torch.randn(T, H, 576, generator=g, device="cuda").to(torch.bfloat16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    slots = ints([0, 1, 2, 3])
    new = [[1 + (29 * i + 53 * k) % 90 for k in range(B)] for i in range(24)]
    rows = [(ints(n), ints([(37 * i + 311 * k) % 1100 for k in range(B)])) for i, n in enumerate(new)]

    def attend(e):
        return rt.mla_prefill(q, latent, None, 512, 64, e.block_tables, e.cu_seqlens_q, e.seq_lens, 90, 1280, bmm1_scale=1 / 24,
                              return_lse=True, window=window, sinks=3)

    def run(wait):
        tables, lens, refs = torch.full((B, 20), -1, dtype=torch.int32, device="cuda"), ints([0] * B), ints([0] * pages)
        rt.extend_pages(tables, lens, slots, ints([1140] * B), refs, page, 4 * 1140)
        start, outs = [t.clone() for t in (tables, lens, refs)], []
        torch.cuda.synchronize()
        for n, keep in rows:
            for t, t0 in zip((tables, lens, refs), start):
                t.copy_(t0)
            e = rt.extend_pages(tables, lens, slots, n, refs, page, T, lens=keep)
            if wait:
                torch.cuda.synchronize()
            outs.append(attend(e))
            if wait:
                torch.cuda.synchronize()
        assert kernels(lambda: attend(e)) == 3
        return outs

    want, got = run(True), run(False)
    assert rt.device_errors() == 0
    for n, (a, al), (b, bl) in zip(new, want, got):
        assert torch.equal(a[: sum(n)], b[: sum(n)]) and torch.equal(al[: sum(n)], bl[: sum(n)])
