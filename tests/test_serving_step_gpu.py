"""GPU: the serving operators together (chunked prefill, fork, decode, free, compact), and in a
captured CUDA graph."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from glm53_flash_dual_dgx_spark_b200 import serving_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,prompt", [(64, 700), (16, 130), (5, 64)])
def test_serving_loop(heads, prompt):
    got = serving_step.run(heads=heads, prompt=prompt, steps=2)
    assert got["device_errors"] == 0
    assert got["fork_equals_parent"] and got["compaction_keeps_outputs"]
    assert got["shared_pages"] == prompt // 64
    assert got["highest_page"] == got["live_pages"] - 1
    assert not torch.isnan(got["out"]).any()


def test_chunks_and_one_pass_agree():
    """A prompt prefilled in chunks gives each token what one pass over the whole prompt gives it:
    the same scores, keys and probabilities, summed in tiles cut elsewhere (fp32 sums of the same
    fp16 products: the outputs' bf16 rounding, 2^-8, may differ by one step)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, H = 1000, 16
    pool = torch.zeros(20, 64, 288, dtype=torch.uint8, device="cuda")
    rt.write_nvfp4(torch.randn(1280, 512, generator=g, device="cuda").to(torch.bfloat16), pool, torch.arange(1280, device="cuda"))
    table = torch.randperm(20, generator=g, device="cuda")[None].int()
    q = torch.randn(n, H, 576, generator=g, device="cuda").to(torch.bfloat16)
    one = lambda lo, hi: rt.mla_prefill(q[lo:hi], pool, None, 512, 64, table, torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"),  # noqa: E731
                                        torch.tensor([hi], dtype=torch.int32, device="cuda"), hi - lo, hi, bmm1_scale=1 / 24)
    whole = one(0, n).float()
    parts = torch.cat([one(lo, min(lo + 300, n)) for lo in range(0, n, 300)]).float()
    assert bool(((whole - parts).abs() <= 2.0 ** -7 * whole.abs() + 2.0 ** -9).all())
    assert rt.device_errors() == 0


def test_prefill_in_a_cuda_graph_follows_the_lengths_on_the_device():
    g = torch.Generator(device="cuda").manual_seed(5)
    H = 32
    pool = torch.zeros(40, 64, 288, dtype=torch.uint8, device="cuda")
    rt.write_nvfp4(torch.randn(2560, 512, generator=g, device="cuda").to(torch.bfloat16), pool, torch.arange(2560, device="cuda"))
    tables = torch.randperm(40, generator=g, device="cuda").view(2, 20).int()
    q = torch.randn(10, H, 576, generator=g, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda")
    seq = torch.tensor([900, 1200], dtype=torch.int32, device="cuda")
    out = torch.empty(10, H, 512, dtype=torch.bfloat16, device="cuda")
    call = lambda: rt.mla_prefill(q, pool, None, 512, 64, tables, cu, seq, 8, 1280, out=out, bmm1_scale=1 / 24)  # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
    for lens, starts in (([900, 1200], [0, 4, 10]), ([33, 1280], [0, 1, 9]), ([1280, 5], [0, 8, 10])):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(torch.tensor(starts, dtype=torch.int32))
        torch.cuda.synchronize()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got[: starts[-1]], out[: starts[-1]])
        assert bool((got[starts[-1]:] == 7.0).all())
    assert rt.device_errors() == 0


def test_every_operator_in_one_graph():
    """Rotate, write, attend, fork, free and compact as one captured graph: a replay gives what the
    calls give, also after larger calls on the same stream have grown the buffers there."""
    g = torch.Generator(device="cuda").manual_seed(9)
    pages, page, H = 64, 16, 16
    randn = lambda *n: torch.randn(*n, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    latent = torch.zeros(pages, page, 288, dtype=torch.uint8, device="cuda")
    rt.write_nvfp4(randn(pages * page, 512), latent, torch.arange(pages * page, device="cuda"))
    rope = randn(pages, page, 64)
    tables = torch.full((8, 16), -1, dtype=torch.int32, device="cuda")
    tables[0, :7] = torch.arange(20, 27, dtype=torch.int32)
    tables[1, :3] = torch.arange(50, 53, dtype=torch.int32)
    seq = torch.tensor([101, 37, 0, 0, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[20:27], refs[50:53] = 1, 1
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    src, dst, ended, cu = ints(0, 1, 0), ints(2, 3, 4), ints(1), ints(0, 3, 4)
    cos_sin = rt.rope_cos_sin(256).cuda()
    positions = torch.tensor([98, 99, 100, 36], device="cuda")
    slots = torch.tensor([26 * 16 + 2, 26 * 16 + 3, 26 * 16 + 4, 52 * 16 + 4], device="cuda")
    q, k_pe, x = randn(4, H, 576), randn(4, 64), randn(4, 2, 128)
    state = [latent, rope, tables, seq, refs, q]
    start = [t.clone() for t in state]
    out = torch.empty(4, H, 512, dtype=torch.bfloat16, device="cuda")
    turned = torch.empty_like(x)

    def calls():
        rt.apply_rope(x, positions, cos_sin, out=turned)
        rt.write_nvfp4_rope_rotated(k_pe, rope, slots, positions, cos_sin, q_pe=q[..., 512:])
        rt.mla_prefill(q, latent, None, 512, 64, tables[:2], cu, seq[:2], 3, 256, out=out, rope_cache=rope, bmm1_scale=1 / 24)
        rt.fork_pages([latent, rope], tables, seq, src, dst, refs)
        rt.free_pages(tables, seq, ended, refs)
        return rt.compact_pages([latent, rope], tables, refs)

    def reset():
        for t, t0 in zip(state, start):
            t.copy_(t0)
        out.zero_()
        turned.zero_()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        live = int(calls())
        want = [t.clone() for t in state + [out, turned]]
        reset()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            count = calls()
        rt.mla_prefill(randn(900, H, 576), latent, None, 512, 64, tables[:1], ints(0, 900), ints(100), 900, 256)
        rt.compact_pages([torch.zeros(9000, 16, 288, dtype=torch.uint8, device="cuda")], ints(3).view(1, 1),
                         torch.zeros(9000, dtype=torch.int32, device="cuda").index_fill(0, torch.tensor([3], device="cuda"), 1))
        for _ in range(2):
            reset()
            graph.replay()
            s.synchronize()
            assert int(count) == live == 12      # 7 + 1 + 1 of the first prompt, 3 of the fork of the second
            for a, b in zip(state + [out, turned], want):
                assert torch.equal(a, b)
    assert rt.device_errors() == 0
