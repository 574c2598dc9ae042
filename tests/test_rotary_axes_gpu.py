"""GPU: rotary positions with several axes against the formula in 64 bits.

Pair i of token t turns by the angle at (positions[axis[i], t], i) of the table.  A rotated value is two
products and a sum in fp32, (|a c| + |b s|) (3 * 2^-24), and one rounding to the type, half a step."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def exact(x, pos, table, axes, offset, interleaved, inverse, most):
    """(values, their tolerance before the rounding) of x [T, H, D] float64; bad tokens stay."""
    r = table.shape[1]
    y, slack = x.clone(), torch.zeros_like(x)
    good = ((pos >= 0) & (pos < most)).all(0)
    for i, a in enumerate(axes):
        p = pos[a].clamp(0, most - 1)
        c, s = table[p, i][:, None], table[p, r // 2 + i][:, None] * (-1.0 if inverse else 1.0)
        da, db = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + r // 2 + i)
        u, v = x[:, :, da], x[:, :, db]
        g = good[:, None]
        y[:, :, da], y[:, :, db] = torch.where(g, u * c - v * s, u), torch.where(g, v * c + u * s, v)
        slack[:, :, da] = ((u * c).abs() + (v * s).abs()) * 3 * 2.0 ** -24
        slack[:, :, db] = ((v * c).abs() + (u * s).abs()) * 3 * 2.0 ** -24
    return y, slack


def close(got, y, slack, dtype):
    eps = HALF_STEP[dtype]
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 2.0 ** -134)          # half the smallest step
    assert bool(((got.double().cpu() - y).abs() <= slack * (1 + eps) + eps * y.abs() + tiny).all())


def inputs(T, H, D, r, A, seed, dtype, most=500):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g).to(dtype)
    pos = torch.randint(0, most, (A, T), generator=g)
    return g, x, pos, rt.rope_cos_sin(most, r)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,H,D,r,offset,A,dealt", [
    (1, 1, 64, 64, 0, 3, False), (16, 64, 576, 64, 512, 3, True), (33, 5, 128, 128, 0, 2, False), (7, 3, 192, 32, 160, 4, True),
    (130, 2, 256, 256, 0, 3, True), (5, 4, 80, 20, 60, 2, True), (9, 1, 33, 6, 1, 3, False), (3, 7, 16, 16, 0, 1, False), (4, 2, 2, 2, 0, 4, False),
])
def test_axes_match_the_formula(T, H, D, r, offset, A, dealt, interleaved, dtype):
    g, x, pos, table = inputs(T, H, D, r, A, T + r, dtype)
    half = r // 2
    sections = [half // A + (1 if a < half % A else 0) for a in range(A)]
    axes = rt.rope_axes(sections, r, dealt=dealt)
    for inverse, index in ((False, torch.int32), (True, torch.int64)):
        out = rt.apply_rope(x.cuda(), pos.to(index).cuda(), table.cuda(), rope_offset=offset, interleaved=interleaved, inverse=inverse, axes=axes)
        y, slack = exact(x.double(), pos, table.double(), axes, offset, interleaved, inverse, table.shape[0])
        close(out, y, slack, dtype)
        keep = torch.ones(D, dtype=torch.bool)
        keep[offset:offset + r] = False
        assert torch.equal(out.cpu()[..., keep], x[..., keep])
    same = x.cuda()
    assert rt.apply_rope(same, pos.cuda(), table.cuda(), rope_offset=offset, interleaved=interleaved, inverse=True, out=same, axes=axes) is same
    assert torch.equal(same, out)
    assert rt.device_errors() == 0


def test_axes_that_agree_give_the_same_bits_as_one():
    for dtype in HALF_STEP:
        for interleaved in (True, False):
            _, x, pos, table = inputs(50, 6, 192, 64, 3, 1, dtype)
            x, table, one = x.cuda(), table.cuda(), pos[0].cuda()
            a = rt.apply_rope(x, one, table, interleaved=interleaved)
            for axes in (rt.rope_axes((8, 12, 12)), rt.rope_axes((8, 12, 12), dealt=True), list(range(3)) * 10 + [2, 2]):
                assert torch.equal(a, rt.apply_rope(x, one.expand(3, -1), table, interleaved=interleaved, axes=axes))


def test_the_gradient_of_the_rotation():
    """inverse is the transpose: <R x, y> = <x, R^T y>, and the finite difference of a linear map is
    the map (fp32: 64 * 12 sums of products, 2^-24 each)."""
    g, x, pos, table = inputs(13, 12, 64, 64, 3, 5, torch.float32)
    axes, table, p = rt.rope_axes((10, 11, 11), dealt=True), table.cuda(), pos.int().cuda()
    y = torch.randn(13, 12, 64, generator=g)
    rx = rt.apply_rope(x.cuda(), p, table, axes=axes).cpu().double()
    ry = rt.apply_rope(y.cuda(), p, table, inverse=True, axes=axes).cpu().double()
    a, b = rx * y.double(), x.double() * ry
    assert bool(((a.sum((1, 2)) - b.sum((1, 2))).abs() <= 4 * 2.0 ** -24 * (rx.abs() * y.double().abs() + x.double().abs() * ry.abs()).sum((1, 2)) * 3).all())
    step = 2.0 ** -6
    moved = rt.apply_rope((x + step * y).cuda(), p, table, axes=axes).cpu().double()
    forward = rt.apply_rope(y.cuda(), p, table, axes=axes).cpu().double()
    slack = (4 * 2.0 ** -24) * (rx.abs() + moved.abs() + 2 * (x.abs().double() + y.abs().double()).amax()) / step
    assert bool((((moved - rx) / step - forward).abs() <= slack).all())


def test_bad_positions_and_views():
    """A position outside the table on any axis leaves its token as it is, flagged; positions and x as
    strided views."""
    g, x, pos, table = inputs(20, 4, 128, 64, 3, 9, torch.bfloat16)
    pos[1, 3], pos[2, 7], pos[0, 11] = -1, 500, 1 << 40
    axes = rt.rope_axes((16, 8, 8))
    wide = torch.zeros(20, 6, 160, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:5, 16:144] = x.cuda()
    out = rt.apply_rope(wide[:, 1:5, 16:144], pos.cuda(), table.cuda(), rope_offset=32, axes=axes)
    assert rt.device_errors() == _lib.DEVERR_BAD_INDEX
    y, slack = exact(x.double(), pos, table.double(), axes, 32, True, False, 500)
    close(out, y, slack, torch.bfloat16)
    for t in (3, 7, 11):
        assert torch.equal(out[t].cpu(), x[t])
    pos = pos.clamp(0, 499)
    y, slack = exact(x.double(), pos, table.double(), axes, 32, True, False, 500)
    rows = torch.zeros(5, 40, dtype=torch.int32, device="cuda")
    rows[1:4, 7:27] = pos.cuda()
    columns = torch.zeros(20, 5, dtype=torch.int64, device="cuda")
    columns[:, 1:4] = pos.T.cuda()
    shifted = torch.zeros(20 * 4 * 128 + 3, dtype=torch.bfloat16, device="cuda")
    shifted[3:] = x.cuda().flatten()
    for xs in (x.cuda(), shifted[3:].view(20, 4, 128)):
        for ps in (rows[1:4, 7:27], columns[:, 1:4].T):
            close(rt.apply_rope(xs, ps, table.cuda(), rope_offset=32, axes=axes), y, slack, torch.bfloat16)
    assert rt.device_errors() == 0
    assert rt.apply_rope(x[:0].cuda(), rows[:3, :0], table.cuda(), axes=axes).shape == (0, 4, 128)


@pytest.mark.parametrize("T,H,interleaved,aligned", [(1, 64, True, True), (37, 3, False, True), (700, 16, True, True), (9, 5, True, False), (9, 0, False, False)])
def test_rotated_keys_into_the_cache(T, H, interleaved, aligned):
    g = torch.Generator().manual_seed(T)
    table = rt.rope_cos_sin(900)
    pos = torch.randint(0, 900, (3, T), generator=g)
    axes = rt.rope_axes((16, 8, 8), dealt=True)
    k, q = torch.randn(T, 64, generator=g).to(torch.bfloat16), torch.randn(T, max(H, 1), 64, generator=g).to(torch.bfloat16)
    shift = 64 if aligned else 61
    wide = torch.zeros(T, 192, dtype=torch.bfloat16, device="cuda")
    wide[:, shift:shift + 64] = k.cuda()
    qw = torch.zeros(T, max(H, 1), 192, dtype=torch.bfloat16, device="cuda")
    qw[..., shift:shift + 64] = q.cuda()
    qo = torch.zeros(T, max(H, 1), 192, dtype=torch.bfloat16, device="cuda")
    cache = torch.full((50, 16, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    slots = torch.randperm(800, generator=g)[:T]
    slots[2::5] = -1
    got = rt.write_nvfp4_rope_rotated(wide[:, shift:shift + 64], cache, slots.cuda(), pos.int().cuda(), table.cuda(),
                                      q_pe=qw[..., shift:shift + 64] if H else None, q_out=qo[..., shift:shift + 64] if H else None,
                                      interleaved=interleaved, axes=axes)
    assert rt.device_errors() == 0
    y, slack = exact(k.double()[:, None], pos, table.double(), axes, 0, interleaved, False, 900)
    live = slots >= 0
    close(cache.view(-1, 64)[slots[live].cuda()][:, None], y[live], slack[live], torch.bfloat16)
    rest = torch.ones(800, dtype=torch.bool)
    rest[slots[live]] = False
    assert bool((cache.view(-1, 64).cpu()[rest] == 3.0).all())
    if H:
        y, slack = exact(q.double(), pos, table.double(), axes, 0, interleaved, False, 900)
        close(got, y, slack, torch.bfloat16)
        assert not qo[..., :shift].any() and not qo[..., shift + 64:].any()
        again = rt.write_nvfp4_rope_rotated(wide[:, shift:shift + 64], cache, slots.cuda(), pos.int().cuda(), table.cuda(),
                                            q_pe=qw[..., shift:shift + 64], interleaved=interleaved, axes=axes)
        assert torch.equal(again, got) and torch.equal(qw[..., shift:shift + 64], got)


def test_a_graph_follows_the_positions():
    g, x, pos, table = inputs(40, 8, 64, 64, 3, 2, torch.bfloat16)
    xs, p, table, axes = x.cuda(), pos.int().cuda(), table.cuda(), rt.rope_axes((8, 12, 12))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rt.apply_rope(xs, p, table, axes=axes)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = rt.apply_rope(xs, p, table, axes=axes)
        p.copy_(pos.flip(1).int())
        graph.replay()
        s.synchronize()
    assert torch.equal(out, rt.apply_rope(xs, pos.flip(1).int().cuda(), table, axes=axes))


@pytest.mark.parametrize("change,error,word", [
    (dict(positions=lambda: torch.zeros(4, dtype=torch.int32, device="cuda")), ValueError, "axes, 4"),
    (dict(positions=lambda: torch.zeros(3, 5, dtype=torch.int32, device="cuda")), ValueError, "axes, 4"),
    (dict(positions=lambda: torch.zeros(5, 4, dtype=torch.int32, device="cuda")), ValueError, "at most 4"),
    (dict(positions=lambda: torch.zeros(3, 4, device="cuda")), TypeError, "int64 or int32"),
    (dict(positions=torch.zeros(3, 4, dtype=torch.int32)), ValueError, "CUDA"),
    (dict(axes=None), ValueError, "entries for 4|axes"),
    (dict(axes=(0, 1, 2)), ValueError, "32 numbers"),
    (dict(axes=(3,) * 32), ValueError, "32 numbers"),
    (dict(axes=(-1,) * 32), ValueError, "32 numbers"),
])
def test_refusals(change, error, word):
    args = dict(positions=lambda: torch.zeros(3, 4, dtype=torch.int32, device="cuda"), axes=(0, 1, 2, 2) * 8) | change
    if callable(args["positions"]):
        args["positions"] = args["positions"]()
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(8, 64, device="cuda")
    with pytest.raises(error, match=word):
        rt.apply_rope(x, cos_sin=table, **args)
    with pytest.raises(error, match=word):
        rt.write_nvfp4_rope_rotated(x[:, 0], torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda"),
                                    torch.zeros(4, dtype=torch.int64, device="cuda"), cos_sin=table, **args)


def test_rotated_dims_past_the_limit():
    x = torch.zeros(2, 1, 512, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="256"):
        rt.apply_rope(x, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 258, device="cuda"), axes=(0,) * 129)
