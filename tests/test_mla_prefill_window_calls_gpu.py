"""GPU: windowed chunk attention in each of its forms as a serving loop calls it: replayed from graphs
whose lengths and tables change, on two streams at once, and within a workspace of exactly the size asked for."""
import ctypes

import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_window_forms_gpu import FORMS, device_call, kernels
from test_mla_prefill_window_gpu import CASES, LARGE, Windowed

pytestmark = pytest.mark.gpu
# (and the units of eight parts in a cluster)
ALL = FORMS + [([1] * 15, [1100, 700, 800, 896, 2000] * 3, 64, 1000, 4, 1)]


@pytest.mark.parametrize("new,ctx,H,window,sinks,num", ALL)
def test_replays_follow_lengths_and_tables(new, ctx, H, window, sinks, num):
    p = Windowed(new, ctx, H, 64, True, window, sinks, seed=num)
    B, T = len(new), sum(new)
    cu, seq, tables = torch.zeros(B + 1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda"), p.tables.cuda()
    out, lse = torch.empty(T, H, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(T, H, device="cuda")

    def call():
        lse.copy_(rt.mla_prefill(p.q, p.pool, None, 512, 64, tables, cu, seq, max(new), max(ctx), out=out, bmm1_scale=p.scale,
                                 rope_cache=p.rope, return_lse=True, window=window, sinks=sinks)[1])

    assert kernels(call) == num              # (the copy of lse is none)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
    every = list(range(B))
    for turn, (lens, n) in enumerate(((ctx, new), ([max(c // 2, k) for c, k in zip(ctx, new)], new), ([c * (b % 2) for b, c in zip(every, ctx)], [k * (b % 2) for b, k in zip(every, new)]),
                                      ([c if b == 0 else 1 for b, c in zip(every, ctx)], [1] * B), (ctx[::-1] if len(set(new)) == 1 else ctx, new))):
        perm = torch.randperm(p.pages, generator=torch.Generator().manual_seed(turn)).int()
        p.tables = torch.full_like(p.tables, -1)
        at = 0
        for b, c in enumerate(lens):
            need = -(-c // 64)
            p.tables[b, :need] = perm[at:at + need]
            at += need
        starts = [sum(n[:b]) for b in range(B + 1)]
        seq.copy_(torch.tensor(lens, dtype=torch.int32)), cu.copy_(torch.tensor(starts, dtype=torch.int32)), tables.copy_(p.tables)
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        live = starts[-1]
        assert bool((out[live:] == 7.0).all()) and rt.device_errors() == 0
        got, e = out.clone(), lse.clone()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got[:live], out[:live]) and torch.equal(e[:live], lse[:live])
        q, p.q, p.new, p.ctx = p.q, p.q[:live], n, lens
        p.check(got[:live], e[:live])
        p.q = q


@pytest.mark.parametrize("first", range(len(ALL)))
def test_two_streams_at_once(first):
    """Calls of two forms that overlap: neither's workspace is the other's."""
    pair = [Windowed(*ALL[k][:3], 64, True, *ALL[k][3:5], seed=k) for k in (first, (first + 1) % len(ALL))]
    calls = [device_call(p) for p in pair]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in pair], [[], []]
    for _ in range(20):
        for k, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[k].append(c())
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, want[k][0]) and torch.equal(b, want[k][1]) for a, b in got[k])
    assert rt.device_errors() == 0


@pytest.mark.parametrize("case", [(*c[:3], 64, True, *c[3:5]) for c in ALL] + CASES[::3] + LARGE[::2])
def test_a_workspace_of_the_size_asked_for(case):
    new, ctx, H, page, rope, window, sinks = case
    p = Windowed(*case, trim=True, seed=2)
    need = ctypes.c_size_t(0)
    most = min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1)
    assert _lib.lib().nvfp4kv_mla_prefill_window_workspace_size(len(new), sum(new), H, max(new), max(ctx), *most, ctypes.byref(need)) == _lib.OK
    want, lse = p.run()
    room = torch.full((need.value + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    seq = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    outs = torch.full((sum(new) + 2, H, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    got = rt.mla_prefill(p.q, p.pool, room[4096:4096 + need.value], 512, 64, p.tables.cuda(), cu, seq, max(new), max(ctx), out=outs[1:-1],
                         bmm1_scale=p.scale, rope_cache=p.rope, return_lse=True, window=window, sinks=sinks)
    assert torch.equal(got[0], want) and torch.equal(got[1], lse)
    assert bool((room[:4096] == 0xA5).all()) and bool((room[4096 + need.value:] == 0xA5).all())
    assert need.value == 0 or bool((room[4096:4096 + need.value] != 0xA5).any())
    assert bool((outs[0] == 7.0).all()) and bool((outs[-1] == 7.0).all())
    assert rt.device_errors() == 0
