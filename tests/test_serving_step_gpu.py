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
